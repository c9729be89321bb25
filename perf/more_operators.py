"""Routing, 8-bit integer products and sampling around the MoE layer, as cases that can be timed.

* route, route_grad: the choice of experts from a router's logits and the experts' weights, by softmax or sigmoid
  scores, a bias for balance and groups of experts, and its gradient (mgpt_amd.routing.ExpertRouting);
* linear: a product in 8-bit integers with a scale for each token and each output (mgpt_amd.linear8.I8Linear);
* experts: the layer's SwiGLU experts by such products, on a routing that the caller has made
  (mgpt_amd.moe.MoELayer with weights="i8", forward_routed);
* sample: a token for each row of logits from a given random number, by temperature, top-k, top-p and min-p
  (mgpt_amd.sampling.Sampler).

listed() holds the cases, draw() spreads more of them over the same ranges. With `own` false run() computes the plain
form in elementary torch operations, with `own` true it calls the package's operators.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
LARGEST = torch.finfo(torch.float32).max
INF = float("inf")


def _route(name, op, act, N, E, k, score, bias=False, groups=1, top_groups=1, renorm=True, scale=1.0, masked=False,
           balance=False):
    return {"name": name, "op": op, "act": act, "N": N, "E": E, "k": k, "score": score, "bias": bias,
            "groups": groups, "top_groups": top_groups, "renorm": renorm, "scale": scale, "masked": masked,
            "balance": balance}


def _linear(name, act, N, K, M, bias=False):
    return {"name": name, "op": "linear", "act": act, "N": N, "K": K, "M": M, "bias": bias}


def _experts(name, act, N, C, E, k, H):
    return {"name": name, "op": "experts", "act": act, "N": N, "C": C, "E": E, "k": k, "H": H}


def _sample(name, act, B, V, top_k=0, top_p=1.0, min_p=0.0):
    return {"name": name, "op": "sample", "act": act, "B": B, "V": V, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # a decode step's tokens (cfg5) through a router trained with a bias for balance
        _route("route_decode_f32", "route", "f32", 64, 64, 8, "sigmoid", True),
        # a long prompt over many experts in 8 groups, of which 4 take part
        _route("route_groups_f32", "route", "f32", 32768, 256, 8, "sigmoid", True, 8, 4, True, 2.5),
        # the headline batch (cfg3) in training
        _route("route_grad_f32", "route_grad", "f32", 16384, 16, 2, "softmax"),
        # a ragged batch over an odd number of experts, some of them masked out, with a balance loss
        _route("route_grad_ragged_bf16", "route_grad", "bf16", 40001, 160, 6, "softmax", False, 8, 3, True, 1.0, True,
               True),
        # one token through the head (cfg5's width, an odd vocabulary)
        _linear("linear_token_bf16", "bf16", 1, 2048, 50257),
        # a prompt
        _linear("linear_prompt_bf16", "bf16", 16384, 2048, 8192),
        # a ragged fp32 batch
        _linear("linear_ragged_f32", "f32", 999, 500, 1003, True),
        # a decode step's context (cfg5)
        _experts("experts_decode_bf16", "bf16", 64, 2048, 64, 8, 1408),
        # the headline layer (cfg3)
        _experts("experts_prompt_bf16", "bf16", 16384, 1024, 16, 2, 2816),
        # one sequence's next token
        _sample("sample_one_f32", "f32", 1, 50257, 50, 0.9),
        # a serving batch over a large vocabulary
        _sample("sample_batch_bf16", "bf16", 256, 131072, 0, 0.95, 0.01),
        # a batch that is sampled without restriction, an odd vocabulary
        _sample("sample_open_f32", "f32", 64, 100003),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    """A pass's rough cost in operations: a byte takes the time of about 300."""
    w = work(case)
    return w["flops"] + 300 * w["bytes"]


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        op = rng.choice(("route", "route_grad", "linear", "experts", "sample"))
        act = rng.choice(("f32", "bf16"))
        if op.startswith("route"):
            groups = rng.choice((1, 1, 2, 4, 8))
            E = groups * _log_int(rng, 4 if groups == 1 else 2, 512 // groups)
            score = rng.choice(("softmax", "sigmoid"))
            case = _route("", op, act, _log_int(rng, 1, 65536), E, rng.randint(1, min(8, E)), score, rng.random() < 0.5,
                          groups, rng.randint(1, groups), rng.random() < 0.7, rng.choice((1.0, 2.5)),
                          rng.random() < 0.25, op == "route_grad" and rng.random() < 0.5)
        elif op == "linear":
            # widths of models are round, odd ones have to work as well
            K, M = _log_int(rng, 16, 8192), _log_int(rng, 16, 65536)
            if rng.random() < 0.75:
                K, M = max(64, K // 64 * 64), max(64, M // 64 * 64)
            case = _linear("", act, _log_int(rng, 1, 16384), K, M, rng.random() < 0.5)
        elif op == "experts":
            E = rng.choice((4, 8, 12, 16, 64, 96))
            case = _experts("", act, _log_int(rng, 1, 16384), _log_int(rng, 8, 256) * 8, E, rng.randint(1, min(8, E)),
                            _log_int(rng, 8, 352) * 8)
        else:
            case = _sample("", act, _log_int(rng, 1, 256), _log_int(rng, 100, 262144),
                           rng.choice((0, 0, 1, 20, _log_int(rng, 1, 1000))), rng.choice((1.0, 0.95, 0.5)),
                           rng.choice((0.0, 0.0, 0.05)))
        if _cost(case) <= most[op]:
            del case["name"]
            return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda").mul_(std)


def _int8_rows(x):
    """Rows in 8-bit integers: (rint(x 127 / max|x|), max|x| / 127), the integers from 64 bits, as many values lie next
    to a border between two of them; a row of zeros gives zeros."""
    top = x.abs().amax(-1, keepdim=True)
    q = (x.double() * (127.0 / top.double())).round().float()
    return torch.where(top > 0, q, torch.zeros_like(q)), (top / 127.0).squeeze(-1)


def prepare(case, seed):
    gen = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op.startswith("route"):
        N, E, k, dt = case["N"], case["E"], case["k"], _DT[case["act"]]
        # a token's logits lie around the experts' own offsets, as a trained router's do
        l = _normal(gen, N, E, std=1.5) + _normal(gen, E, std=0.5) - 1
        if case["masked"]:
            l.masked_fill_(torch.rand(N, E, generator=gen, device="cuda") < 0.03, -INF)
        s["l"] = l.to(dt)
        s["b"] = _normal(gen, E, std=0.05) if case["bias"] else None
        s["dw"] = _normal(gen, N, k) if op == "route_grad" else None
        s["ds"] = _normal(gen, E, std=0.01) if case["balance"] else None
        if own:
            from mgpt_amd.routing import ExpertRouting
            s["op"] = ExpertRouting(E, k, score=case["score"], groups=case["groups"], top_groups=case["top_groups"],
                                    group_best=2, renormalise=case["renorm"], scale=case["scale"], act=case["act"])
        return s
    if op == "linear":
        N, K, M, dt = case["N"], case["K"], case["M"], _DT[case["act"]]
        # tokens of different sizes, and a few columns that are much larger than the others
        x = _normal(gen, N, K) * torch.exp(_normal(gen, N, 1, std=0.5))
        s["x"] = (x * torch.exp(_normal(gen, K, std=0.5))).to(dt)
        s["q"] = _normal(gen, M, K, std=32.0).round_().clamp_(-127, 127).to(torch.int8)
        s["sw"] = torch.exp(_normal(gen, M, std=0.3)) * (0.02 / 32)
        s["b"] = _normal(gen, M, std=0.1) if case["bias"] else None
        if own:
            from mgpt_amd.linear8 import I8Linear
            s["op"] = I8Linear(K, M, act=case["act"])
            s["op"].load_quantized(s["q"], s["sw"], bias=s["b"])
        return s
    if op == "experts":
        N, C, E, k, H, dt = case["N"], case["C"], case["E"], case["k"], case["H"], _DT[case["act"]]
        s["x"] = (_normal(gen, N, C) * torch.exp(_normal(gen, C, std=0.3))).to(dt)
        # some experts are chosen more often than others
        score = _normal(gen, N, E) + _normal(gen, E, std=0.3)
        top, idx = score.topk(k, 1)
        s["idx"], s["w"] = idx.int(), torch.softmax(top, 1)
        # the most rows of an expert, which the plain form's batched products are padded to
        s["rows"] = int(torch.bincount(idx.view(-1), minlength=E).max())
        params = [_normal(gen, C, E, std=0.02), torch.zeros(E, device="cuda")]
        for name, a, b in (("g", C, H), ("u", C, H), ("d", H, C)):
            W = _normal(gen, E, a, b, std=1 / math.sqrt(a))
            s["W" + name], s["s" + name] = _int8_rows(W.transpose(1, 2))
            s["W" + name] = s["W" + name].to(torch.int8).contiguous()
            s["b" + name] = _normal(gen, E, b, std=0.05)
            params.append((W, s["b" + name]) if own else None)
        if own:
            from mgpt_amd.moe import MoELayer
            s["op"] = MoELayer(C, H, E, k, act=case["act"], weights="i8")
            s["op"].load_parameters(params[:2] + [t for e in range(E) for W, b in params[2:] for t in (W[e], b[e])])
        return s
    B, V = case["B"], case["V"]
    # the head's logits: a few large ones over a wide floor
    l = _normal(gen, B, V, std=2.0)
    l += 6 * torch.rand(B, V, generator=gen, device="cuda").pow_(64)
    s["l"] = l.to(_DT[case["act"]])
    s["u"] = torch.rand(B, generator=gen, device="cuda")
    # every request of a batch has a temperature of its own, some of them none at all
    s["T"] = 0.6 + 0.6 * torch.rand(B, generator=gen, device="cuda")
    if B > 8:
        s["T"][::16] = 0
    s["k"] = torch.full((B,), case["top_k"], dtype=torch.int32, device="cuda")
    s["p"] = torch.full((B,), case["top_p"], device="cuda")
    s["m"] = torch.full((B,), case["min_p"], device="cuda")
    if own:
        from mgpt_amd.sampling import Sampler
        s["op"] = Sampler(V, act=case["act"])
    return s


# ------------------------------------------------------------- the routing
# An expert whose logit is -inf or NaN takes no part. Experts are chosen by their key: the logit itself where scores are
# compared with each other alone, else the score with the bias, in 64 bits, so that keys next to each other are told
# apart. A group counts by the sum of its two best keys, and ties go to the lowest number.
def _order(key):
    return torch.sort(key, dim=-1, descending=True, stable=True)


def _softmax(l):
    """A row of which every expert is masked has no probabilities: zeros."""
    z = (l - l.amax(1, keepdim=True).clamp(min=-LARGEST)).exp()
    return z / z.sum(1, keepdim=True).clamp(min=1e-30)


def _plain_keys(s):
    case = s["case"]
    l = s["l"].float()
    if not case["bias"] and case["groups"] == 1:
        return torch.where(l.isnan(), torch.full_like(l, -INF), l)
    l = l.double()
    if case["score"] == "softmax":
        key = _softmax(l)
    else:
        key = 1 / (1 + (-l).exp())
    if case["bias"]:
        key = key + s["b"].double()
    return torch.where(l > -INF, key, torch.full_like(key, -INF))


def _plain_scores(s):
    l = s["l"].float()
    if s["case"]["score"] == "sigmoid":
        return 1 / (1 + (-l).exp())
    return _softmax(l)


def _plain_route(s):
    case = s["case"]
    N, E, G = case["N"], case["E"], case["groups"]
    key = _plain_keys(s)
    if G > 1:
        best = _order(key.view(N, G, E // G))[0][:, :, :2]
        some = best[:, :, 0] > -INF
        size = torch.where(best > -INF, best, torch.zeros_like(best)).sum(2)
        size = torch.where(some, size, torch.full_like(size, -INF))
        chosen = torch.zeros_like(size, dtype=torch.bool)
        chosen.scatter_(1, _order(size)[1][:, :case["top_groups"]], True)
        key = torch.where(chosen.repeat_interleave(E // G, 1), key, torch.full_like(key, -INF))
    key, idx = _order(key)
    idx = idx[:, :case["k"]]
    score = _plain_scores(s)
    sel = torch.where(key[:, :case["k"]] > -INF, score.gather(1, idx), torch.zeros(1, device="cuda"))
    D = sel.sum(1, keepdim=True) + 1e-20
    w = sel * case["scale"]
    if case["renorm"]:
        w = w / D
    out = {"idx": idx.int(), "w": w}
    if case["op"] == "route":
        return out
    dw, on = s["dw"], key[:, :case["k"]] > -INF
    d = dw * case["scale"]
    if case["renorm"]:
        d = (d - (d * sel).sum(1, keepdim=True) / D) / D
    ds = torch.zeros_like(score)
    ds.scatter_(1, idx, torch.where(on, d, torch.zeros_like(d)))
    if s["ds"] is not None:
        ds = ds + s["ds"]
    if case["score"] == "sigmoid":
        dl = ds * score * (1 - score)
    else:
        dl = score * (ds - (ds * score).sum(1, keepdim=True))
    out["dl"] = dl.to(s["l"].dtype)
    return out


def _own_route(s):
    idx, w = s["op"].forward(s["l"], bias=s["b"])
    out = {"idx": idx, "w": w}
    if s["case"]["op"] == "route_grad":
        out["dl"] = s["op"].backward(s["l"], idx, w, s["dw"], dscores=s["ds"])
    return out


def _exact_route(s):
    case = s["case"]
    N, E, k, G = case["N"], case["E"], case["k"], case["groups"]
    l = s["l"].double()
    p = torch.softmax(l, 1).nan_to_num(nan=0.0) if case["score"] == "softmax" else torch.sigmoid(l)
    there = ~torch.isneginf(l)
    key = p + (s["b"].double() if case["bias"] else 0)
    key[~there] = -INF
    if G > 1:
        two = key.view(N, G, -1).sort(dim=2, descending=True)[0][:, :, :2]
        size = two[:, :, 0] + (two[:, :, 1].nan_to_num(neginf=0.0) if two.shape[2] > 1 else 0)
        rank = size.sort(dim=1, descending=True, stable=True)[1].argsort(1)
        key = key.masked_fill((rank >= case["top_groups"]).repeat_interleave(E // G, 1), -INF)
    at = key.sort(dim=1, descending=True, stable=True)[1][:, :k]
    on = key.gather(1, at) > -INF
    # the weights as a function of the logits, differentiated by the chain rule: J^T dw
    ps = p.gather(1, at) * on
    total = ps.sum(1, keepdim=True) + 1e-20 if case["renorm"] else torch.ones_like(ps[:, :1])
    w = case["scale"] * ps / total
    out = {"idx": at.int(), "w": w}
    if case["op"] == "route_grad":
        up = s["dw"].double() * on
        g = case["scale"] * up / total
        if case["renorm"]:
            g = g - (up * w).sum(1, keepdim=True) / total * on
        full = torch.zeros_like(p).scatter_add_(1, at, g)
        if s["ds"] is not None:
            full += s["ds"].double()
        if case["score"] == "softmax":
            out["dl"] = p * full - p * (p * full).sum(1, keepdim=True)
        else:
            out["dl"] = full * torch.sigmoid(l) * torch.sigmoid(-l)
    return out


# ------------------------------------------------------- 8-bit products
def _plain_linear(s):
    q, sx = _int8_rows(s["x"].float())
    y = (q @ s["q"].float().t()) * sx[:, None] * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(s["x"].dtype)


def _exact_linear(s):
    x = s["x"].double()
    most = x.abs().amax(1, keepdim=True).clamp(min=1e-300)
    y = torch.round(127 / most * x).mm(s["q"].double().t())
    y = y * (most / 127) * s["sw"].double()[None]
    return y if s["b"] is None else y + s["b"].double()


def _plain_experts(s):
    case = s["case"]
    N, C, E, k, R = case["N"], case["C"], case["E"], case["k"], s["rows"]
    flat = s["idx"].long().view(-1)
    e, order = torch.sort(flat, stable=True)
    counts = torch.zeros(E, dtype=torch.long, device="cuda").scatter_add_(0, flat, torch.ones_like(flat))
    first = counts.cumsum(0) - counts
    slot = e * R + torch.arange(N * k, device="cuda") - first[e]   # each expert's rows, padded to R
    x = torch.zeros(E * R, C, device="cuda").index_copy_(0, slot, s["x"].float()[order // k]).view(E, R, C)

    def product(a, name):
        q, sa = _int8_rows(a)
        W = s["W" + name].float().transpose(1, 2).contiguous()
        return torch.bmm(q, W) * sa[:, :, None] * s["s" + name][:, None] + s["b" + name][:, None]

    g, u = product(x, "g"), product(x, "u")
    o = product(g / (1 + (-g).exp()) * u, "d").view(E * R, C)
    back = torch.empty_like(slot).index_copy_(0, order, slot)
    y = (o[back].view(N, k, C) * s["w"][:, :, None]).sum(1)
    return y.to(s["x"].dtype)


def _exact_experts(s):
    """An expert at a time in 64 bits."""
    case = s["case"]
    y = torch.zeros(case["N"], case["C"], dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        t, j = (s["idx"] == e).nonzero(as_tuple=True)
        if not t.numel():
            continue

        def product(a, name):
            most = a.abs().amax(1).clamp(min=1e-300)
            r = torch.round(a * (127 / most)[:, None]) @ s["W" + name][e].double().t()
            return r * torch.outer(most / 127, s["s" + name][e].double()) + s["b" + name][e].double()

        x = s["x"][t].double()
        o = product(torch.nn.functional.silu(product(x, "g")) * product(x, "u"), "d")
        y.index_add_(0, t, o * s["w"][t, j].double()[:, None])
    return y


# -------------------------------------------------------------- sampling
# Weights are whole numbers, exp((l - max) / T) in units of 2^-40, so that their sums have no order. A temperature of 0
# takes the largest logit. The tokens that stay are the first of the order by logit (ties: the lowest id): top_k of
# them (0: all), of those the ones before which less than top_p of their sum lies, and the ones of at least min_p. The
# token is the first, by id, at which their running sum exceeds u times their sum.
UNITS = 2.0 ** 40


def _plain_sample(s):
    V = s["case"]["V"]
    l = s["l"].float().clamp(max=LARGEST)
    greedy = s["T"] <= 0
    T = torch.where(greedy, torch.ones_like(s["T"]), s["T"])
    k = torch.where(greedy, torch.ones_like(s["k"]), torch.where(s["k"] <= 0, torch.full_like(s["k"], V), s["k"]))
    sl, si = _order(l)
    W = (((sl.double() - sl[:, :1].double()) / T.double()[:, None]).exp() * UNITS).round()
    first = torch.arange(V, device="cuda")[None] < k[:, None]
    Wk = torch.where(first, W, torch.zeros_like(W)).long()
    run = Wk.cumsum(1)
    p = s["p"].double()[:, None]
    keep = first & (((run - Wk).double() < p * run[:, -1:].double()) | (p >= 1))
    keep &= W >= s["m"].double()[:, None] * UNITS
    keep[:, 0] = True
    mine = torch.zeros_like(Wk).scatter_(1, si, torch.where(keep, Wk, torch.zeros_like(Wk)))
    run = mine.cumsum(1)
    total = run[:, -1:]
    at = (run.double() <= s["u"].double()[:, None] * total.double()).sum(1)
    at = torch.minimum(at, (run < total).sum(1))
    z = (l.gather(1, at[:, None]).double() - sl[:, :1].double()).squeeze(1) / T.double()
    return {"token": at.int(), "logp": (z - (total.squeeze(1).double() / UNITS).log()).float()}


def _own_sample(s):
    token, logp = s["op"].forward(s["l"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
    return {"token": token, "logp": logp}


def _exact_sample(s):
    """A row at a time, with probabilities in 64 bits."""
    tokens, logps = [], []
    for r in range(s["case"]["B"]):
        l = s["l"][r].double()
        T, k, p, m, u = (float(s[n][r]) for n in ("T", "k", "p", "m", "u"))
        if T <= 0:
            tokens.append(int((l == l.max()).nonzero()[0]))
            logps.append(0.0)
            continue
        v, i = l.sort(descending=True, stable=True)
        i = i[:int(k)] if k > 0 else i
        w = ((v[:len(i)] - v[0]) / T).exp()
        n = len(i) if p >= 1 else max(1, int((w.cumsum(0) - w < p * w.sum()).sum()))
        i = i[:max(1, min(n, int((w >= m).sum())))]
        ids = i.sort()[0]
        w = ((l[ids] - v[0]) / T).exp()
        n = min(int((w.cumsum(0) <= u * w.sum()).sum()), len(ids) - 1)
        tokens.append(int(ids[n]))
        logps.append(float(w[n].log() - w.sum().log()))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "logp": torch.tensor(logps, dtype=torch.float64)}


def run(s):
    op = s["case"]["op"]
    if op.startswith("route"):
        return _own_route(s) if own else _plain_route(s)
    if op == "linear":
        return s["op"].forward(s["x"]) if own else _plain_linear(s)
    if op == "experts":
        return s["op"].forward_routed(s["x"], s["idx"], s["w"]) if own else _plain_experts(s)
    return _own_sample(s) if own else _plain_sample(s)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("route"):
        return _exact_route(s)
    return {"linear": _exact_linear, "experts": _exact_experts, "sample": _exact_sample}[op](s)


def work(case):
    op = case["op"]
    if op.startswith("route"):
        N, E, k, e = case["N"], case["E"], case["k"], _SIZE[case["act"]]
        bytes_, flops = N * E * e + N * k * 8 + (4 * E if case["bias"] else 0), 10 * N * E
        if op == "route_grad":
            bytes_ += 2 * N * E * e + N * k * 8 + (4 * E if case["balance"] else 0)
            flops += 15 * N * E
        return {"bytes": bytes_, "flops": flops}
    if op == "linear":
        N, K, M, e = case["N"], case["K"], case["M"], _SIZE[case["act"]]
        return {"bytes": N * (K + M) * e + M * K + 4 * M * (2 if case["bias"] else 1), "flops": 2 * N * K * M}
    if op == "experts":
        N, C, E, k, H, e = case["N"], case["C"], case["E"], case["k"], case["H"], _SIZE[case["act"]]
        used = min(E, N * k)
        return {"bytes": used * (3 * C * H + 4 * (4 * H + 2 * C)) + 2 * N * C * e + 8 * N * k, "flops": 6 * N * k * C * H}
    B, V = case["B"], case["V"]
    return {"bytes": B * V * _SIZE[case["act"]] + 28 * B, "flops": 20 * B * V}
