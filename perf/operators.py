"""The work of a training step around the MoE block, as cases that can be timed.

Three operators, each with a plain form in elementary torch operations:

* the language model's loss: softmax cross entropy of x . W^T + b over the
  vocabulary, and its gradients (mgpt_amd.loss.LMLoss);
* one AdamW step over all tensors of a model, with moments in 32 bits or in
  8 bits per value (mgpt_amd.optim.AdamW);
* the norms around a block: its output normalised, gated and added to the
  scaled residual stream, and the sum normalised for the next block, forward
  and backward (mgpt_amd.norm.ResidualNorm).

listed() holds the cases, draw() spreads more of them over the same ranges.
With `own` false run() computes the plain form, with `own` true it calls the
package's operators.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
EPS_NORM = 1e-5
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256   # elements that share the exponents of 8-bit moments


def _loss(name, op, act, N, C, V, bias=True):
    return {"name": name, "op": op, "act": act, "N": N, "C": C, "V": V, "bias": bias}


def _adamw(name, bits, grads, C, H, E, extra=0, copies=False, clip=False):
    return {"name": name, "op": "adamw", "bits": bits, "grads": grads, "C": C, "H": H, "E": E,
            "extra": extra, "copies": copies, "clip": clip}


def _norm(name, op, act, N, C, groups, scale=1.0):
    return {"name": name, "op": op, "act": act, "N": N, "C": C, "groups": groups, "scale": scale}


def listed():
    return [
        # the engine's default batch (cfg1: 16 x 64 tokens) over a byte vocabulary, fp32, a whole training pass
        _loss("loss_grad_default_f32", "loss_grad", "f32", 1024, 128, 256),
        # scoring the 64-token context of a sampling loop (cfg5's width) over an odd-sized vocabulary
        _loss("loss_context_bf16", "loss", "bf16", 64, 2048, 50257),
        # evaluation: the loss alone, a batch of the mid-size block (cfg2's tokens)
        _loss("loss_eval_bf16", "loss", "bf16", 8192, 1024, 65536, False),
        # a ragged fp32 batch of a small model
        _loss("loss_grad_ragged_f32", "loss_grad", "f32", 999, 500, 8003),
        # the headline training step's batch (cfg3) with the gradients of its head
        _loss("loss_grad_bf16", "loss_grad", "bf16", 16384, 1024, 32000, False),
        # the engine's default layer (cfg1): 50 tensors, small ones among them
        _adamw("adamw_default", 32, "f32", 128, 512, 8),
        # the headline layer (cfg3): 98 tensors, 139 million parameters
        _adamw("adamw_headline", 32, "f32", 1024, 2816, 16, 0, False, True),
        # the same with 8-bit moments, bf16 gradients and the bf16 weights refreshed
        _adamw("adamw8_headline", 8, "bf16", 1024, 2816, 16, 0, True, True),
        # a small ragged layer in 8 bits
        _adamw("adamw8_ragged", 8, "f32", 250, 333, 6, 1001),
        # a decode step's rows (cfg5) through the norms
        _norm("norm_decode_bf16", "norm", "bf16", 64, 2048, 1),
        # training, one gate for all tokens (cfg3's rows)
        _norm("norm_grad_bf16", "norm_grad", "bf16", 16384, 1024, 1, 0.5),
        # training at the fine-grained layer's width (cfg4), a gate for each of 64 sequences
        _norm("norm_grad_wide_bf16", "norm_grad", "bf16", 32768, 2048, 64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    """A pass's rough cost in bf16 operations: fp32 products run at a
    sixteenth of the bf16 rate, a byte takes the time of about 300."""
    w = work(case)
    return w["flops"] * (16 if case.get("act") == "f32" else 1) + 300 * w["bytes"]


def draw(rng):
    most = {}
    for c in listed():
        kind = c["op"].split("_")[0]
        most[kind] = max(most.get(kind, 0), _cost(c))
    while True:
        kind = rng.choice(("loss", "adamw", "norm"))
        if kind == "loss":
            act = rng.choice(("f32", "bf16", "bf16"))
            c = _log_int(rng, 16, 512 if act == "f32" else 4096)
            # widths of models are round, odd ones have to work as well
            c = c if rng.random() < 0.25 else max(64, c // 64 * 64)
            case = _loss("", rng.choice(("loss", "loss_grad", "loss_grad")), act,
                         _log_int(rng, 1, 4096 if act == "f32" else 16384), c,
                         _log_int(rng, 16, 16384 if act == "f32" else 131072), rng.random() < 0.5)
        elif kind == "adamw":
            bits = rng.choice((32, 8))
            case = _adamw("", bits, rng.choice(("f32", "bf16")), _log_int(rng, 16, 2048),
                          _log_int(rng, 16, 2816), _log_int(rng, 1, 64), rng.choice((0, _log_int(rng, 1, 10000))),
                          rng.random() < 0.5, rng.random() < 0.5)
        else:
            groups = rng.choice((1, 1, _log_int(rng, 1, 64)))
            case = _norm("", rng.choice(("norm", "norm_grad")), rng.choice(("f32", "bf16")),
                         groups * _log_int(rng, 1, 32768 // groups), _log_int(rng, 16, 8192), groups,
                         rng.choice((1.0, 0.5)))
            case["C"] = case["C"] if rng.random() < 0.25 else max(64, case["C"] // 64 * 64)
        if _cost(case) <= most[kind]:
            del case["name"]
            return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda").mul_(std)


def _sizes(case):
    """Elements of the layer's tensors: the router's, and per expert gate, up
    and down with their biases; `extra` is one more tensor (a norm's scale)."""
    C, H, E = case["C"], case["H"], case["E"]
    return [C * E, E] + [C * H, H, C * H, H, H * C, C] * E + ([case["extra"]] if case["extra"] else [])


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _views(flat, sizes):
    """A tensor per entry of sizes, each at a multiple of BLOCK elements."""
    out, at = [], 0
    for n in sizes:
        out.append(flat[at:at + n])
        at += _padded(n)
    return out


def _holes(sizes):
    """The positions of the padded elements between those tensors."""
    mask = torch.ones(sum(_padded(n) for n in sizes), dtype=torch.bool)
    for v in _views(mask, sizes):
        v.fill_(False)
    return mask.cuda()


def prepare(case, seed):
    gen = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op.startswith("loss"):
        N, C, V, dt = case["N"], case["C"], case["V"], _DT[case["act"]]
        s["x"] = _normal(gen, N, C).to(dt)
        s["W"] = _normal(gen, V, C, std=0.02).to(dt)
        s["b"] = _normal(gen, V, std=0.1) if case["bias"] else None
        t = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
        # one token in sixteen is padding and has no target
        pad = torch.randint(0, 16, (N,), generator=gen, device="cuda") == 0
        s["t"] = torch.where(pad, torch.full_like(t, -1), t)
        if own:
            from mgpt_amd.loss import LMLoss
            s["op"] = LMLoss(C, V, act=case["act"])
        return s
    if op == "adamw":
        sizes = _sizes(case)
        n = sum(_padded(k) for k in sizes)
        hole = _holes(sizes)
        s["p"] = _normal(gen, n, std=0.02).masked_fill_(hole, 0)
        # gradients of very different sizes from block to block, as layers have them
        size = torch.exp(_normal(gen, n // BLOCK, 1) - 7)
        g = (_normal(gen, n // BLOCK, BLOCK) * size).view(-1).masked_fill_(hole, 0)
        s["g"] = g.to(_DT[case["grads"]])
        s["clip"] = torch.full((1,), 0.7, device="cuda") if case["clip"] else None
        s["copy"] = s["p"].to(torch.bfloat16) if case["copies"] else None
        s["step"] = 100
        m = (_normal(gen, n // BLOCK, BLOCK) * size * 0.3).view(-1).masked_fill_(hole, 0)
        v = (g * 0.8).square().view(-1)
        if case["bits"] == 8:
            s["m"], s["me"] = _encode_m(m)
            s["v"], s["ve"] = _encode_v(v, 0)
        else:
            s["m"], s["v"] = m, v
        if own:
            from mgpt_amd.optim import AdamW
            s["op"] = AdamW(_views(s["p"], sizes), lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                            state_bits=case["bits"], copies=_views(s["copy"], sizes) if case["copies"] else None)
            s["grads"] = _views(s["g"], sizes)
            s["op"].step_count = s["step"]
            s["op"].m.copy_(s["m"])
            s["op"].v.copy_(s["v"])
            if case["bits"] == 8:
                s["op"].m_exp.copy_(s["me"])
                s["op"].v_exp.copy_(s["ve"])
        return s
    N, C, G, dt = case["N"], case["C"], case["groups"], _DT[case["act"]]
    s["x"] = _normal(gen, N, C, std=3.0).to(dt)
    s["h"] = (_normal(gen, N, C) * torch.exp(_normal(gen, N, 1))).to(dt)
    s["post"] = 1 + _normal(gen, C, std=0.1)
    s["gate"] = _normal(gen, G, C, std=0.5)
    s["pre"] = 1 + _normal(gen, C, std=0.1)
    if op == "norm_grad":
        s["dout"] = _normal(gen, N, C).to(dt)
        s["dy"] = _normal(gen, N, C).to(dt)
    if own:
        from mgpt_amd.norm import ResidualNorm
        s["op"] = ResidualNorm(C, act=case["act"], eps=EPS_NORM, residual_scale=case["scale"])
    return s


# --------------------------------------------------------------- the loss
def _plain_loss(s):
    x, W, t = s["x"].float(), s["W"].float(), s["t"].long()
    logits = x @ W.t()
    if s["b"] is not None:
        logits = logits + s["b"]
    top = logits.amax(1, keepdim=True)
    lse = (top + (logits - top).exp().sum(1, keepdim=True).log()).squeeze(1)
    valid = (t >= 0) & (t < W.shape[0])
    picked = logits.gather(1, t.clamp(0, W.shape[0] - 1)[:, None]).squeeze(1)
    loss = torch.where(valid, lse - picked, torch.zeros_like(lse))
    count = valid.sum()
    mean = torch.stack([loss.double().sum() / count.clamp(min=1), count.double()]).float()
    out = {"loss": loss, "lse": lse, "mean": mean}
    if s["case"]["op"] == "loss":
        return out
    # d(mean loss) / d(logits) = (softmax - onehot) / count on the valid rows
    d = (logits - lse[:, None]).exp()
    d.scatter_add_(1, t.clamp(0, W.shape[0] - 1)[:, None], -torch.ones_like(lse)[:, None])
    d = d * (valid / count.clamp(min=1))[:, None]
    out["dx"] = (d @ W).to(s["x"].dtype)
    out["dW"] = (d.t() @ x).to(s["W"].dtype)
    if s["b"] is not None:
        out["db"] = d.sum(0)
    return out


def _own_loss(s):
    loss, lse, mean = s["op"].forward(s["x"], s["W"], s["t"], bias=s["b"])
    out = {"loss": loss, "lse": lse, "mean": mean}
    if s["case"]["op"] == "loss_grad":
        dx, dW, db = s["op"].backward(s["x"], s["W"], s["t"], lse, bias=s["b"])
        out["dx"], out["dW"] = dx, dW
        if db is not None:
            out["db"] = db
    return out


def _exact_loss(s):
    """Rows at a time in 64 bits, the probabilities from the logits' own sums."""
    case = s["case"]
    W = s["W"].double()
    V, N = W.shape[0], s["x"].shape[0]
    t = s["t"].long()
    has = (t > -1) & (t < V)
    count = int(has.sum())
    share = 1.0 / max(count, 1)
    rows = max(1, min(N, (1 << 27) // V))
    losses, lses, dxs = [], [], []
    dW = torch.zeros_like(W) if case["op"] == "loss_grad" else None
    db = torch.zeros(V, dtype=torch.float64, device="cuda")
    for r in range(0, N, rows):
        x = s["x"][r:r + rows].double()
        z = x @ W.t()
        if s["b"] is not None:
            z += s["b"].double()
        lse = torch.logsumexp(z, 1)
        tr, hr = t[r:r + rows], has[r:r + rows]
        at = torch.arange(x.shape[0], device="cuda")[hr]
        loss = torch.zeros_like(lse)
        loss[hr] = lse[hr] - z[at, tr[hr]]
        losses.append(loss)
        lses.append(lse)
        if dW is not None:
            p = torch.softmax(z, 1)
            p[at, tr[hr]] -= 1
            p[~hr] = 0
            p *= share
            dxs.append(p @ W)
            dW += p.t() @ x
            db += p.sum(0)
    loss = torch.cat(losses)
    out = {"loss": loss, "lse": torch.cat(lses),
           "mean": torch.stack([loss.sum() * share, torch.tensor(float(count), dtype=torch.float64, device="cuda")])}
    if dW is not None:
        out["dx"], out["dW"] = torch.cat(dxs), dW
        if s["b"] is not None:
            out["db"] = db
    return out


# ---------------------------------------------------------- the optimizer
# Moments in 8 bits: 256 neighbours share one power of two.  The first moment
# is an e4m3 number, rounded to nearest even, times 2^(e - 134), e the biased
# exponent of the block's largest magnitude (at least 16).  The second moment
# is never negative, spans far more and moves by a thousandth a step: five
# bits of exponent and three of fraction, of which the largest value's
# exponent is 30, and rounded up or down at random, so that what is below a
# step's rounding counts on average; a value above zero is never held as zero.
def _exponent(x):
    return x.view(torch.int32) >> 23


def _encode_m(m):
    b = m.view(-1, BLOCK)
    e = _exponent(b.abs().amax(1)).clamp(min=16)
    scale = ((261 - e) << 23).view(torch.float32)[:, None]             # 2^(134 - e)
    return (b * scale).to(torch.float8_e4m3fn).view(-1), e.to(torch.uint8)


def _decode_m(q, e):
    scale = ((e.int() - 7) << 23).view(torch.float32)[:, None]           # 2^(e - 134)
    return (q.view(-1, BLOCK).float() * scale).view(-1)


def _random16(n, step):
    """A 16-bit number for each element: half of a mixed 32-bit counter."""
    pair = torch.arange((n + 1) // 2, device="cuda")
    x = (pair ^ ((step * 0x9E3779B9) & 0xFFFFFFFF)) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    return torch.stack([x & 0xFFFF, x >> 16], 1).view(-1)[:n].int()


def _encode_v(v, step):
    b = v.view(-1, BLOCK)
    e = (_exponent(b.amax(1)) + 1).clamp(min=32)
    code = ((b.view(torch.int32) + (_random16(v.numel(), step).view(-1, BLOCK) << 4)) >> 20) - ((e - 31) << 3)[:, None]
    code = torch.where(b > 0, code.clamp(1, 254), torch.zeros_like(code))
    return code.to(torch.uint8).view(-1), e.to(torch.uint8)


def _decode_v(q, e):
    c = q.view(-1, BLOCK).int()
    bits = ((e.int() - 31) << 23)[:, None] + (c << 20)
    return torch.where(c > 0, bits, torch.zeros_like(bits)).view(torch.float32).view(-1)


def _f32(x):
    return torch.tensor(x, dtype=torch.float32).item()


def _plain_adamw(s):
    case = s["case"]
    s["step"] += 1
    t = s["step"]
    b1, b2, lr, eps, wd = _f32(BETA1), _f32(BETA2), _f32(LR), _f32(EPS), _f32(DECAY)
    c1, c2 = _f32(1 / (1 - b1 ** t)), _f32(1 / (1 - b2 ** t))
    a1, a2, shrink = _f32(1 - b1), _f32(1 - b2), _f32(lr * wd)
    g = s["g"].float()
    if s["clip"] is not None:
        g = g * s["clip"]
    if case["bits"] == 8:
        m, v = _decode_m(s["m"], s["me"]), _decode_v(s["v"], s["ve"])
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * a1
    v = v * b2 + (g * a2) * g
    p = s["p"] - s["p"] * shrink
    p = p - ((m * c1) * lr) / ((v * c2).sqrt() + eps)
    s["p"].copy_(p)
    out = {"p": s["p"]}
    if case["bits"] == 8:
        s["m"], s["me"] = _encode_m(m)
        s["v"], s["ve"] = _encode_v(v, t)
        out["me"], out["ve"] = s["me"], s["ve"]
    else:
        s["m"], s["v"] = m, v
    out["m"], out["v"] = s["m"], s["v"]
    if s["copy"] is not None:
        s["copy"].copy_(p)
        out["copy"] = s["copy"]
    return out


def _own_adamw(s):
    o = s["op"]
    o.step(s["grads"], grad_scale=s["clip"])
    out = {"p": s["p"], "m": o.m, "v": o.v}
    if s["case"]["bits"] == 8:
        out["me"], out["ve"] = o.m_exp, o.v_exp
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    return out


def _exact_adamw(s):
    """The step in 64 bits from the moments as they are held; what is held in
    8 bits afterwards depends on roundings and has no such value."""
    case = s["case"]
    t = s["step"] + 1
    b1, b2, lr, eps, wd = (float(_f32(k)) for k in (BETA1, BETA2, LR, EPS, DECAY))
    g = s["g"].double() * (float(s["clip"]) if s["clip"] is not None else 1.0)
    if case["bits"] == 8:
        m = (s["m"].float().double().view(-1, BLOCK) * torch.exp2(s["me"].double() - 134)[:, None]).view(-1)
        c = s["v"].double().view(-1, BLOCK)
        v = (1 + torch.remainder(c, 8) / 8) * torch.exp2(torch.floor(c / 8) + s["ve"].double()[:, None] - 158)
        v = torch.where(c > 0, v, torch.zeros_like(v)).view(-1)
    else:
        m, v = s["m"].double(), s["v"].double()
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).addcmul_(g, g, value=1 - b2)
    p = s["p"].double() * (1 - lr * wd)
    p.sub_(lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps))
    small = case["bits"] == 8
    out = {"p": p, "m": None if small else m, "v": None if small else v}
    if small:
        out["me"], out["ve"] = None, None
    if s["copy"] is not None:
        out["copy"] = p
    return out


# --------------------------------------------------------------- the norms
def _plain_norm(s):
    case = s["case"]
    N, C, G, a = case["N"], case["C"], case["groups"], case["scale"]
    x, h = s["x"].float(), s["h"].float()
    gate = s["gate"].repeat_interleave(N // G, 0)
    rh = (h.square().mean(1, keepdim=True) + EPS_NORM).rsqrt()
    n = h * rh
    u = n * s["post"]
    o = x * a + u * gate
    ro = (o.square().mean(1, keepdim=True) + EPS_NORM).rsqrt()
    z = o * ro
    dt = s["x"].dtype
    out = {"out": o.to(dt), "y": (z * s["pre"]).to(dt), "rh": rh.squeeze(1), "ro": ro.squeeze(1)}
    if case["op"] == "norm":
        return out
    dy = s["dy"].float()
    q = dy * s["pre"]
    do = s["dout"].float() + ro * (q - z * (q * z).mean(1, keepdim=True))
    du = do * gate
    dn = du * s["post"]
    out["dx"] = (do * a).to(dt)
    out["dh"] = (rh * (dn - n * (dn * n).mean(1, keepdim=True))).to(dt)
    out["dpost"] = (du * n).sum(0)
    out["dgate"] = (do * u).view(G, N // G, C).sum(1)
    out["dpre"] = (dy * z).sum(0)
    return out


def _own_norm(s):
    o = s["op"]
    out, y, rh, ro = o.forward(s["x"], s["h"], gamma_post=s["post"], gate=s["gate"], gamma_pre=s["pre"])
    r = {"out": out, "y": y, "rh": rh, "ro": ro}
    if s["case"]["op"] == "norm_grad":
        g = o.backward(s["x"], s["h"], s["dout"], s["dy"], rh, ro, gamma_post=s["post"], gate=s["gate"],
                       gamma_pre=s["pre"])
        r["dx"], r["dh"], r["dpost"], r["dgate"], r["dpre"] = g
    return r


def _exact_norm(s):
    """A gate's rows at a time in 64 bits."""
    case = s["case"]
    N, C, G, a = case["N"], case["C"], case["groups"], case["scale"]
    R = N // G
    post, pre = s["post"].double(), s["pre"].double()
    keep = {k: [] for k in ("out", "y", "rh", "ro", "dx", "dh", "dgate")}
    dpost = torch.zeros(C, dtype=torch.float64, device="cuda")
    dpre = torch.zeros_like(dpost)
    for i in range(G):
        rows = slice(i * R, (i + 1) * R)
        x, h, gate = s["x"][rows].double(), s["h"][rows].double(), s["gate"][i].double()
        rh = 1 / torch.sqrt((h * h).sum(1) / C + EPS_NORM)
        o = a * x + gate * post * h * rh[:, None]
        ro = 1 / torch.sqrt((o * o).sum(1) / C + EPS_NORM)
        keep["out"].append(o)
        keep["y"].append(pre * o * ro[:, None])
        keep["rh"].append(rh)
        keep["ro"].append(ro)
        if case["op"] == "norm_grad":
            dy = s["dy"][rows].double()
            k = dy * pre
            do = s["dout"][rows].double() + k * ro[:, None] - o * (ro ** 3 * (k * o).sum(1) / C)[:, None]
            w = do * gate * post
            keep["dx"].append(a * do)
            keep["dh"].append(w * rh[:, None] - h * (rh ** 3 * (w * h).sum(1) / C)[:, None])
            t = (do * h * rh[:, None]).sum(0)
            keep["dgate"].append((t * post)[None])
            dpost += t * gate
            dpre += (dy * o * ro[:, None]).sum(0)
    names = ["out", "y", "rh", "ro"] + (["dx", "dh", "dgate"] if case["op"] == "norm_grad" else [])
    out = {k: torch.cat(keep[k]) for k in names}
    if case["op"] == "norm_grad":
        out["dpost"], out["dpre"] = dpost, dpre
    return out


def run(s):
    op = s["case"]["op"]
    if op.startswith("loss"):
        return _own_loss(s) if own else _plain_loss(s)
    if op == "adamw":
        return _own_adamw(s) if own else _plain_adamw(s)
    return _own_norm(s) if own else _plain_norm(s)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    return _exact_loss(s) if op.startswith("loss") else _exact_adamw(s) if op == "adamw" else _exact_norm(s)


def work(case):
    op = case["op"]
    if op.startswith("loss"):
        N, C, V, e = case["N"], case["C"], case["V"], _SIZE[case["act"]]
        b = 4 * V if case["bias"] else 0
        bytes_, flops = (N + V) * C * e + b + N * 12, 2 * N * C * V
        if op == "loss_grad":
            # the logits again (they are not kept), d(x) and d(W)
            bytes_ += 2 * (N + V) * C * e + 2 * b + N * 8
            flops *= 4
        return {"bytes": bytes_, "flops": flops}
    if op == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 * (1 + 1 / BLOCK)
        return {"bytes": n * (8 + _SIZE[case["grads"]] + state + (2 if case["copies"] else 0)), "flops": 14 * n}
    N, C, e = case["N"], case["C"], _SIZE[case["act"]]
    gains = 4 * C * (2 + case["groups"])
    bytes_, flops = 4 * N * C * e + gains + 8 * N, 10 * N * C
    if op == "norm_grad":
        bytes_ += 6 * N * C * e + 2 * gains + 8 * N
        flops += 30 * N * C
    return {"bytes": bytes_, "flops": flops}
