"""mgpt_adamw_step (mgpt_amd.optim.AdamW) against the step's formula in 64 bits
and, bit for bit, in the engine's order of fp32 operations (Tensor::adamw_step,
utils/Tensor.cpp:683-701); 8-bit moments against the format's definition,
restated here on the CPU.

Tolerances against 64 bits, u = 2^-24 (half a step of fp32):
  m: the scaled gradient, two products and a sum are 4 roundings of terms no
     larger than A = |b1 m| + |a1 g|: 4 u A.
  v: 5 roundings of non-negative terms: 5 u v, and the square of the scaled
     gradient's own rounding, 2 u: 8 u v.
  p: the decay and the two differences round |p| at most 3 times; the quotient
     carries m's error, half of v's and 6 roundings of its own: 16 u times
     lr c1 A / (sqrt(v c2) + eps).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F = np.float32
LR, B1, B2, EPS, WD = F(1e-2), F(0.9), F(0.999), F(1e-8), F(0.1)
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


def make(params, **kw):
    from mgpt_amd.optim import AdamW
    return AdamW(params, lr=float(LR), betas=(float(B1), float(B2)), eps=float(EPS), weight_decay=float(WD), **kw)


def blocks(n):
    return (n + 255) // 256


def flat_slices(sizes):
    out, at = [], 0
    for n in sizes:
        out.append(slice(at, at + n))
        at += blocks(n) * 256
    return out, at


def step_f32(p, g, m, v, t, scale):
    """The engine's order, every operation rounded to float32."""
    one = F(1)
    c1 = F(1.0 / (1.0 - float(B1) ** t))
    c2 = F(1.0 / (1.0 - float(B2) ** t))
    g = g * F(scale)
    m = B1 * m + (one - B1) * g
    v = B2 * v + ((one - B2) * g) * g
    p = p - F(LR * WD) * p
    p = p - (LR * (m * c1)) / (np.sqrt(v * c2) + EPS)
    return p, m, v


def check_f64(p0, g, m0, v0, t, scale, p1, m1, v1):
    p, g, m, v = (np.asarray(a, np.float64) for a in (p0, g, m0, v0))
    g = g * float(F(scale))
    b1, b2, lr = float(B1), float(B2), float(LR)
    amp = np.abs(b1 * m) + np.abs((1 - b1) * g)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    c1, c2 = 1 / (1 - b1 ** t), 1 / (1 - b2 ** t)
    den = np.sqrt(v * c2) + float(EPS)
    ref = p * (1 - lr * float(WD)) - lr * c1 * m / den
    tiny = 1e-44   # products below fp32's smallest number
    assert (np.abs(m1 - m) <= 4 * U * amp + tiny).all()
    assert (np.abs(v1 - v) <= 8 * U * v + tiny).all()
    assert (np.abs(p1 - ref) <= 3 * U * np.maximum(np.abs(p), np.abs(ref)) + 16 * U * lr * c1 * amp / den).all()


def gradients(rng, sizes, bf16):
    gs = [(rng.standard_normal(n) * 10.0 ** rng.uniform(-4, 1)).astype(F) for n in sizes]
    t = [torch.from_numpy(g).cuda() for g in gs]
    if bf16:
        t = [x.bfloat16() for x in t]
        gs = [x.float().cpu().numpy() for x in t]
    return gs, t


SIZES = [[1], [256], [257, 1, 0, 255, 4096], [5000, 3, 70001, 4097], [17] * 233]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("bf16,scale,copies", [(False, None, False), (True, 0.37, True)])
def test_fp32_moments(sizes, bf16, scale, copies):
    rng = np.random.default_rng(5)
    ps = [rng.standard_normal(n).astype(F) for n in sizes]
    params = [torch.from_numpy(p.copy()).cuda() for p in ps]
    cp = [torch.zeros(n, dtype=torch.bfloat16, device="cuda") for n in sizes] if copies else None
    opt = make(params, copies=cp)
    sl, _ = flat_slices(sizes)
    ms = [np.zeros(n, F) for n in sizes]
    vs = [np.zeros(n, F) for n in sizes]
    gs_dev = None if scale is None else torch.full((1,), scale, device="cuda")
    for t in range(1, 4):
        gs, gt = gradients(rng, sizes, bf16)
        opt.step(gt, grad_scale=gs_dev)
        torch.cuda.synchronize()
        M, V = opt.m.cpu().numpy(), opt.v.cpu().numpy()
        for i, s in enumerate(sl):
            p1 = params[i].cpu().numpy()
            check_f64(ps[i], gs[i], ms[i], vs[i], t, 1.0 if scale is None else scale, p1, M[s], V[s])
            p, ms[i], vs[i] = step_f32(ps[i], gs[i], ms[i], vs[i], t, 1.0 if scale is None else scale)
            assert np.array_equal(M[s], ms[i]) and np.array_equal(V[s], vs[i]) and np.array_equal(p1, p), (t, i)
            ps[i] = p
            if copies:
                assert torch.equal(cp[i], params[i].bfloat16())
    # the room after a tensor's end stays zero
    mask = np.ones(M.shape, bool)
    for s in sl:
        mask[s] = False
    assert not M[mask].any() and not V[mask].any()


# ------------------------------------------------------ moments in 8 bits
E4M3 = None


def e4m3_values():
    """The 128 non-negative e4m3 numbers (the last is NaN), from the format."""
    c = np.arange(128)
    e, f = c >> 3, c & 7
    v = np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))
    return v


def encode_m(m):
    """codes, exponents of [blocks, 256] float32, nearest even by search."""
    vals = e4m3_values()[:127]
    fin = np.where(np.isfinite(m), np.abs(m), 0).astype(F)
    e = np.maximum(fin.max(1).view(np.int32) >> 23, 16)
    x = m.astype(np.float64) * 2.0 ** (134.0 - e[:, None])
    a = np.abs(np.where(np.isfinite(x), x, 0))
    hi = np.clip(np.searchsorted(vals, a), 1, 126)
    lo = hi - 1
    dl, dh = a - vals[lo], vals[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(a == 0, 0, c) | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), c, 127).astype(np.uint8), e.astype(np.uint8)


def decode_m(c, e):
    vals = e4m3_values()
    vals[127] = np.nan
    v = vals[c & 127] * np.where(c & 128, -1.0, 1.0)
    return (v * 2.0 ** (np.maximum(e.astype(np.float64), 16) - 134)[:, None]).astype(F)


def hash32(x):
    x = x.astype(np.uint64)
    k = np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & k
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B)) & k
    return x ^ (x >> np.uint64(16))


def encode_v(v, step):
    nb = v.shape[0]
    fin = np.where(np.isfinite(v), v, 0).astype(F)
    e = np.maximum((fin.max(1).view(np.int32) >> 23) + 1, 32).astype(np.int64)
    h = hash32(np.arange(nb * 128, dtype=np.uint64) ^ np.uint64((step * 0x9E3779B9) & 0xFFFFFFFF))
    r = np.stack([h & np.uint64(0xFFFF), h >> np.uint64(16)], 1).reshape(nb, 256).astype(np.int64)
    bits = fin.view(np.int32).astype(np.int64)
    c = np.maximum(((bits + (r << 4)) >> 20) - ((e - 31) << 3)[:, None], 1)
    return np.where(np.isfinite(v), np.where(fin > 0, c, 0), 255).astype(np.uint8), e.astype(np.uint8)


def decode_v(c, e):
    bits = ((np.maximum(e.astype(np.int64), 32) - 31) << 23)[:, None] + (c.astype(np.int64) << 20)
    v = bits.astype(np.int32).view(F).copy()
    v[c == 0] = 0
    v[c == 255] = np.nan
    return v


def pad_blocks(xs):
    return np.concatenate([np.pad(x, (0, blocks(x.size) * 256 - x.size)) for x in xs]).reshape(-1, 256)


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("bf16", [False, True])
def test_8bit_moments(sizes, bf16):
    rng = np.random.default_rng(6)
    ps = [rng.standard_normal(n).astype(F) for n in sizes]
    params = [torch.from_numpy(p.copy()).cuda() for p in ps]
    opt = make(params, state_bits=8)
    nb = sum(blocks(n) for n in sizes)
    cm, cv = np.zeros((nb, 256), np.uint8), np.zeros((nb, 256), np.uint8)
    em = ev = np.zeros(nb, np.uint8)
    P = pad_blocks(ps)
    for t in range(1, 5):
        gs, gt = gradients(rng, sizes, bf16)
        if t == 3 and sizes[0] > 100:   # gradients whose squares leave the range of a block's exponents
            gs[0][:40] *= F(1e-18)
            gs[0][40:50] = 0
            gt[0] = torch.from_numpy(gs[0]).cuda().to(gt[0].dtype)
            gs[0] = gt[0].float().cpu().numpy()
        opt.step(gt)
        torch.cuda.synchronize()
        P, m, v = step_f32(P, pad_blocks(gs), decode_m(cm, em), decode_v(cv, ev), t, 1.0)
        cm, em = encode_m(m)
        cv, ev = encode_v(v, t)
        got = [opt.m.view(torch.uint8), opt.v, opt.m_exp, opt.v_exp]
        got = [g.cpu().numpy() for g in got]
        assert np.array_equal(got[2], em) and np.array_equal(got[3], ev)
        # (a zero's sign is not part of the format's meaning)
        a, b = got[0].reshape(-1, 256), cm
        assert np.array_equal(np.where(a == 128, 0, a), np.where(b == 128, 0, b)), t
        assert np.array_equal(got[1].reshape(-1, 256), cv), t
        sl, _ = flat_slices(sizes)
        for i, s in enumerate(sl):
            assert np.array_equal(params[i].cpu().numpy(), P.reshape(-1)[s]), (t, i)


def test_8bit_second_moment_follows_its_average():
    """A constant gradient's second moment tends to g^2 although each step
    moves it by less than half a code: within three deviations of the mean of
    2048 elements.  A step's rounding is unbiased with variance at most
    (q / 2)^2, q = v / 8 the code's step, and the errors decay by b2 a step, so
    v's deviation is at most (v / 16) / sqrt(1 - b2^2)."""
    n, steps = 2048, 400
    p = torch.zeros(n, device="cuda")
    opt = make([p], state_bits=8)
    g = torch.full((n,), 0.25, device="cuda")
    for _ in range(steps):
        opt.step([g])
    v = decode_v(opt.v.cpu().numpy().reshape(-1, 256), opt.v_exp.cpu().numpy()).astype(np.float64)
    want = 0.0625 * (1 - float(B2) ** steps)
    sd = want / 16 / np.sqrt(1 - float(B2) ** 2) / np.sqrt(n)
    assert abs(v.mean() - want) <= 3 * sd, (v.mean(), want, sd)


def test_values_that_are_not_finite_stay_where_they_are():
    n = 512
    for bits in (32, 8):
        clean = torch.ones(n, device="cuda")
        p = clean.clone()
        half = torch.full((n,), 0.5, device="cuda")
        g = half.clone()
        g[3], g[300] = float("nan"), float("inf")
        a, b = make([clean], state_bits=bits), make([p], state_bits=bits)
        for first, opt in ((half, a), (g, b)):
            opt.step([first])
            opt.step([half])
        bad = torch.tensor([3, 300], device="cuda")
        ok = torch.ones(n, dtype=torch.bool, device="cuda")
        ok[bad] = False
        assert torch.isnan(p[bad]).all()
        assert torch.equal(p[ok], clean[ok])


@pytest.mark.parametrize("bits", [32, 8])
def test_views_at_odd_addresses(bits):
    """Parameters, gradients and copies that are not aligned to vectors give the
    bits of aligned ones, and their neighbours stay."""
    rng = np.random.default_rng(8)
    n = 9000
    p0, g0 = rng.standard_normal(n).astype(F), rng.standard_normal(n).astype(F)
    ref = torch.from_numpy(p0).cuda()
    a = make([ref], state_bits=bits)
    a.step([torch.from_numpy(g0).cuda()])
    for off in (1, 2, 3):
        buf = torch.full((n + 8,), 7.0, device="cuda")
        gbuf = torch.full((n + 8,), 9.0, device="cuda")
        cbuf = torch.full((n + 8,), 5.0, dtype=torch.bfloat16, device="cuda")
        p, g, c = buf[off:off + n], gbuf[off:off + n], cbuf[off:off + n]
        p.copy_(torch.from_numpy(p0))
        g.copy_(torch.from_numpy(g0))
        b = make([p], state_bits=bits, copies=[c])
        b.step([g])
        assert torch.equal(p, ref) and torch.equal(b.state, a.state) and torch.equal(c, ref.bfloat16())
        assert (buf[:off] == 7).all() and (buf[off + n:] == 7).all()
        assert (cbuf[:off] == 5).all() and (cbuf[off + n:] == 5).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradient_leaves_a_tensor(bits):
    p = [torch.ones(300, device="cuda"), torch.ones(300, device="cuda")]
    opt = make(p, state_bits=bits)
    g = torch.ones(300, device="cuda")
    opt.step([g, g])
    before, state = p[0].clone(), opt.m.clone()
    opt.step([None, g])
    assert torch.equal(p[0], before) and torch.equal(opt.m[:512].view(torch.uint8), state[:512].view(torch.uint8))
    assert not torch.equal(p[1], before)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_on(bits):
    """A step captured with its number on the device, replayed, gives the bits
    of eager steps, with eager work between the replays and on another stream."""
    rng = np.random.default_rng(9)
    p0 = rng.standard_normal(5000).astype(F)
    gs = [torch.from_numpy(rng.standard_normal(5000).astype(F)).cuda() for _ in range(4)]
    ref = torch.from_numpy(p0).cuda()
    a = make([ref], state_bits=bits)
    p = torch.from_numpy(p0).cuda()
    g = torch.zeros_like(p)
    b = make([p], state_bits=bits, device_step=True)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            b.step([g])
    torch.cuda.synchronize()
    for gi in gs:
        a.step([gi])
        g.copy_(gi)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, ref) and torch.equal(a.state, b.state)


def test_parameters_keep_their_memory():
    """Memory assigned to a parameter later may have any size, type or device:
    refused, and nothing is written."""
    p = torch.nn.Parameter(torch.ones(600, device="cuda"), requires_grad=False)
    c = torch.zeros(600, dtype=torch.bfloat16, device="cuda")
    opt = make([p], copies=[c])
    g = torch.ones(600, device="cuda")
    opt.step([g])
    was, held = p.data, p.clone()
    for other in (p.data.clone(), p.data.bfloat16(), p.data[1:], p.data.cpu()):
        p.data = other
        with pytest.raises(ValueError, match="memory"):
            opt.step([g])
    p.data = was
    assert torch.equal(p, held) and opt.step_count == 1
    opt.step([g])
    assert not torch.equal(p, held) and torch.equal(c, p.bfloat16())


def test_a_refused_step_is_not_counted():
    from mgpt_amd.capi import MoEError
    p = torch.ones(300, device="cuda")
    ref = p.clone()
    a, b = make([ref]), make([p], device_step=True)
    g = torch.ones(300, device="cuda")
    lr, b.lr = b.lr, float("nan")
    with pytest.raises(MoEError):
        b.step([g])
    b.lr = lr
    a.step([g])
    b.step([g])
    assert torch.equal(p, ref) and b.step_count == 1
