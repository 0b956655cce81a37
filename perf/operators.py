"""What the layer-norm and expert-routing operators are measured on: their cases, inputs, plain forms and exact values.

``run`` computes a case either in its plain form (elementary torch operations) or, with ``own`` set, through the public
calls of ``d2dmoe_amd.ops``.

Layer norm of the rows of ``h`` (``h = x``, or ``h = x + residual`` rounded to the storage type, which is then an output:
the residual stream that the block hands on), over the width D::

    m = sum_d h_d / D        v = sum_d (h_d - m)^2 / D        r = 1 / sqrt(v + eps)        n_d = (h_d - m) r
    out_d = n_d weight_d + bias_d

and backward, for the gradient g of ``out`` and the gradient s of the residual stream::

    u_d = g_d weight_d       grad_d = r (u_d - mean(u) - n_d mean(u n)) + s_d
    grad_weight_d = sum over rows of g_d n_d               grad_bias_d = sum over rows of g_d

Expert routing of a row of logits z (E experts, k of them chosen)::

    s = softmax(z) or 1 / (1 + exp(-z))      the scores
    c = s + bias                             what the choice goes by (z itself without a bias and without sums of scores)
    groups: the E experts in equal runs; a run's score is its largest c, or the sum of its two largest; the best runs stay
    chosen: the k largest c that remain, ties to the lowest index; experts with z = -inf are never chosen, and a row with a
            NaN among its c chooses nothing; places left over hold index -1 and weight 0
    w = scale s, or scale s / sum of the chosen s when renormalised       routing[e] = w at the chosen experts, else 0

and backward, for the gradient q of the weights (of ``routing`` at the chosen experts, or of the weights by place)::

    softmax:  dz_j = scale s_j (q_j [chosen] - sum_i q_i s_i)             renormalised, p = w / scale: w_j (q_j - sum_i q_i p_i)
    sigmoid:  dz_j = scale q_j s_j (1 - s_j)                              renormalised: w_j (1 - s_j) (q_j - sum_i q_i p_i)
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------ cases
def _norm(name, rows, width, dtype, residual, params="same", train=False, bias=True):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "params": params, "train": train, "bias": bias}


def _route(name, tokens, experts, k, dtype, scoring, renormalise, balance=False, groups=1, kept_groups=1,
           group_score="top2", scale=1.0, masked=False, train="no"):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "scoring": scoring,
            "renormalise": renormalise, "balance": balance, "groups": groups, "kept_groups": kept_groups,
            "group_score": group_score, "scale": scale, "masked": masked, "train": train}


def listed():
    return [
        # one generated token of GPT-2 small: the norm between attention and the expert layer, with the residual added
        _norm("norm 1x768", 1, 768, "bf16", True),
        # sixteen generated tokens at the width of the gated layer, float32 parameters
        _norm("norm 16x2048", 16, 2048, "bf16", True, params="f32"),
        # a batch of 256 images of ViT-B, the headline layer's input
        _norm("norm 50432x768", 50432, 768, "bf16", True),
        # a width that no vector load divides, float32, no bias (the bias=False models)
        _norm("norm f32 3001x1001", 3001, 1001, "f32", False, bias=False),
        # a training step of GPT-2 small's batch: 16 sequences of 1024 tokens
        _norm("norm train 16384x768", 16384, 768, "bf16", True, train=True),
        # a ragged packed batch at GPT-2 large's width, float16, no residual (the model's last norm)
        _norm("norm train 4097x1280", 4097, 1280, "f16", False, train=True),
        # the largest: a wide model's training batch with float32 parameters
        _norm("norm train 32768x4096", 32768, 4096, "bf16", True, params="f32", train=True),
        # one generated token: 128 experts, two of them
        _route("route 1x128", 1, 128, 2, "bf16", "softmax", True),
        # the headline layer's tokens and experts, eight of them each
        _route("route 50432x128", 50432, 128, 8, "bf16", "softmax", True),
        # 256 experts in 8 groups of which 4 are kept, sigmoid scores and a balance bias
        _route("route groups 16384x256", 16384, 256, 8, "f32", "sigmoid", True, balance=True, groups=8, kept_groups=4, scale=2.5),
        # a training step of GPT-2 small's batch, softmax weights as they are
        _route("route train 16384x128", 16384, 128, 8, "bf16", "softmax", False, train="routing"),
        # a ragged, padded batch with experts switched off, 60 experts, float16, trained through the compact weights
        _route("route train 3001x60", 3001, 60, 6, "f16", "sigmoid", True, balance=True, masked=True, train="weights"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if rng.random() < 0.5:
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        rows = _log_int(rng, 1, max(1, min(65536, (32768 * 4096 // (2 if dtype == "f32" else 1)) // width)))
        case = _norm("", rows, width, dtype, rng.random() < 0.6, rng.choice(("same", "f32")), rng.random() < 0.5, rng.random() < 0.8)
    else:
        experts = rng.choice((8, 16, 24, 32, 48, 60, 64, 96, 128, 160, 192, 256, 320, 512))
        groups = rng.choice([g for g in (1, 1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
        kept = 1 if groups == 1 else rng.randint(1, groups)
        k = min(rng.choice((1, 2, 4, 6, 8, 8, 12)), experts // groups * kept)
        balance = groups > 1 or rng.random() < 0.4
        train = rng.choice(("no", "routing", "weights"))
        # (a single renormalised weight is constant: nothing is trained through it)
        renormalise = rng.random() < 0.6 and (k > 1 or train == "no")
        case = _route("", _log_int(rng, 1, (1 << 23) // experts), experts, k, dtype, rng.choice(("softmax", "sigmoid")),
                      renormalise, balance, groups, kept, rng.choice(("top2", "max")), rng.choice((1.0, 2.5)),
                      rng.random() < 0.3, train)
    del case["name"]
    return case


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        p = 4 if case["params"] == "f32" else e
        vectors = d * p * (2 if case["bias"] else 1)
        tensors = 4 if case["residual"] else 2                    # x (residual) -> out (h)
        flops = 8 * n * d
        nbytes = tensors * n * d * e + vectors
        if case["train"]:
            nbytes += (3 if case["residual"] else 2) * n * d * e + vectors   # g (s) -> grad; the vectors' gradients
            flops += 16 * n * d
        return {"bytes": nbytes, "flops": flops}
    n, x, k = case["tokens"], case["experts"], case["k"]
    nbytes = 2 * n * x * e + 8 * n * k + (4 * x if case["balance"] else 0)   # logits -> routing, indices and weights
    flops = n * x * (6 + k)
    if case["train"] != "no":
        nbytes += n * x * e + (n * x * e if case["train"] == "routing" else 4 * n * k)
        flops += 6 * n * x
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        pt = torch.float32 if case["params"] == "f32" else t
        # residual streams have a few channels far larger than the others, and a mean that is not zero
        channel = torch.where(torch.rand(d, generator=gen, device=DEV) < 0.01, 12.0, 1.0)
        state = {"case": case, "x": (normal(n, d) * channel + 0.3).to(t),
                 "residual": (normal(n, d) * 0.5).to(t) if case["residual"] else None,
                 "weight": (1.0 + 0.1 * normal(d)).to(pt), "bias": (0.1 * normal(d)).to(pt) if case["bias"] else None,
                 "eps": 1e-5}
        if case["train"]:
            state["grad_out"] = normal(n, d).to(t)
            state["grad_sum"] = normal(n, d).to(t) if case["residual"] else None
        return state
    n, e, k = case["tokens"], case["experts"], case["k"]
    logits = normal(n, e) * 1.5 + normal(e) * 0.5                 # experts differ in popularity
    if case["masked"]:
        logits[:, torch.rand(e, generator=gen, device=DEV) < 0.1] = -math.inf      # experts that are switched off
        logits[torch.rand(n, generator=gen, device=DEV) < 0.05] = -math.inf        # padding: rows that go nowhere
    state = {"case": case, "logits": logits.to(t), "balance": normal(e) * 0.05 if case["balance"] else None}
    if case["train"] == "routing":
        state["grad"] = normal(n, e).to(t)
    elif case["train"] == "weights":
        state["grad"] = normal(n, k)
    return state


def run(state):
    if state["case"]["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_route(state) if own else _plain_route(state)


# -------------------------------------------------------------------------------------------------- the public calls
def _own_norm(s):
    from d2dmoe_amd import ops
    train = s["case"]["train"]
    out, total, mean, rstd = ops.layer_norm(s["x"], s["weight"], s["bias"], s["eps"], s["residual"], want_stats=train)
    if not train:
        return {"out": out, "sum": total}
    grad, grad_weight, grad_bias = ops.layer_norm_backward(s["grad_out"], s["x"] if total is None else total, s["weight"],
                                                           mean, rstd, s["grad_sum"], want_bias=s["bias"] is not None)
    return {"out": out, "sum": total, "grad": grad, "grad_weight": grad_weight, "grad_bias": grad_bias}


def _own_route(s):
    from d2dmoe_amd import ops
    c = s["case"]
    routing, indices, weights, _ = ops.route_topk(s["logits"], c["k"], c["scoring"], s["balance"], c["groups"], c["kept_groups"],
                                                  c["group_score"], c["renormalise"], c["scale"])
    found = {"routing": routing, "indices": indices, "weights": weights}
    if c["train"] != "no":
        by = "grad_routing" if c["train"] == "routing" else "grad_weights"
        found["grad"] = ops.route_topk_backward(s["logits"], indices, c["scoring"], c["renormalise"], c["scale"], **{by: s["grad"]})
    return found


# --------------------------------------------------------------------------------------------------- the plain forms
def _plain_norm(s):
    x, w, b = s["x"], s["weight"].float(), s["bias"]
    total = None if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    h = (x if total is None else total).float()
    mean = h.mean(dim=1, keepdim=True)
    centred = h - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + s["eps"])
    n = centred * rstd
    out = n * w if b is None else n * w + b.float()
    found = {"out": out.to(x.dtype), "sum": total}
    if s["case"]["train"]:
        g = s["grad_out"].float()
        u = g * w
        grad = rstd * (u - u.mean(dim=1, keepdim=True) - n * (u * n).mean(dim=1, keepdim=True))
        if s["grad_sum"] is not None:
            grad = grad + s["grad_sum"].float()
        found["grad"] = grad.to(x.dtype)
        found["grad_weight"] = (g * n).sum(dim=0).to(s["weight"].dtype)
        found["grad_bias"] = None if b is None else g.sum(dim=0).to(b.dtype)
    return found


def _plain_choice(z, c, balance):
    """What the choice goes by, in 64 bits: neighbours in it lie closer together than 32 bits of a score tell apart."""
    z = z.double()
    bad = torch.isnan(z)
    if c["scoring"] == "softmax":
        bad = bad | (z == math.inf)
    if balance is not None or (c["groups"] > 1 and c["group_score"] == "top2"):
        if c["scoring"] == "softmax":
            top = z.amax(dim=1, keepdim=True)
            e = torch.exp(z - torch.where(torch.isfinite(top), top, 0.0))
            by = e / e.sum(dim=1, keepdim=True)
        else:
            by = 1.0 / (1.0 + torch.exp(-z))
        if balance is not None:
            by = by + balance.double()
    else:
        by = z
    by = torch.where(z == -math.inf, -math.inf, by) + 0.0         # + 0.0: the two zeros are one value
    bad = (bad | torch.isnan(by)).any(dim=1, keepdim=True)
    return torch.where(bad, -math.inf, by)


def _plain_route(s):
    z, c, k = s["logits"], s["case"], s["case"]["k"]
    n, e = z.shape
    by = _plain_choice(z, c, s["balance"])
    if c["groups"] > 1:
        runs = by.view(n, c["groups"], -1)
        best = torch.sort(runs, dim=2, descending=True).values[..., :2]
        of_run = best[..., 0]
        if c["group_score"] == "top2" and best.size(2) == 2:
            of_run = of_run + torch.where(best[..., 1] == -math.inf, 0.0, best[..., 1])
        order = torch.sort(of_run, dim=1, descending=True, stable=True).indices[:, :c["kept_groups"]]
        stays = torch.zeros(n, c["groups"], dtype=torch.bool, device=z.device).scatter_(1, order, True)
        by = torch.where(stays.unsqueeze(2), runs, -math.inf).view(n, e)
    sorted_by, order = torch.sort(by, dim=1, descending=True, stable=True)
    there = sorted_by[:, :k] > -math.inf
    place = torch.where(there, order[:, :k], 0)
    zf = z.float()
    at = torch.where(there, zf.gather(1, place), -math.inf)
    if c["scoring"] == "softmax":
        top = (at if c["renormalise"] else zf).amax(dim=1, keepdim=True)
        top = torch.where(torch.isfinite(top), top, 0.0)
        score = torch.exp(at - top)
        whole = score if c["renormalise"] else torch.exp(zf - top)
    else:
        low = at.clamp(max=0.0)
        top = low.amax(dim=1, keepdim=True) if c["renormalise"] else torch.zeros_like(low[:, :1])
        score = torch.exp(low - torch.where(torch.isfinite(top), top, 0.0)) / (1.0 + torch.exp(-at.abs()))
        whole = score
    share = score / whole.sum(dim=1, keepdim=True) if c["renormalise"] or c["scoring"] == "softmax" else score
    share = torch.where(there, share, 0.0)
    weights = c["scale"] * share
    target = torch.where(there, place, e)                         # places left over go to a column that is dropped
    routing = torch.zeros(n, e + 1, device=z.device).scatter_(1, target, weights)[:, :e].to(z.dtype)
    found = {"routing": routing, "indices": torch.where(there, place, -1).int(), "weights": weights}
    if c["train"] != "no":
        q = s["grad"].float()
        q = torch.where(there, q.gather(1, place) if c["train"] == "routing" else q, 0.0)
        d = weights * q
        if c["renormalise"]:                                      # a common part of q has no effect: the first place's goes first
            q = torch.where(there, q - q[:, :1], 0.0)
            d = weights * (q - (share * q).sum(dim=1, keepdim=True))
        if c["scoring"] == "sigmoid":
            d = torch.where(there, d / (1.0 + torch.exp(at)), 0.0)      # 1 - s
        d = torch.zeros(n, e + 1, device=z.device).scatter_(1, target, d)[:, :e]
        if c["scoring"] == "softmax" and not c["renormalise"]:
            some = there.any(dim=1, keepdim=True)
            p = torch.where(some, torch.exp(zf - top) / whole.sum(dim=1, keepdim=True), 0.0)
            d = d - p * (weights * q).sum(dim=1, keepdim=True)
        found["grad"] = d.to(z.dtype)
    return found


# ------------------------------------------------------------------------------------------------------ exact values
def exact(case, seed):
    """From the definitions in 64 bits; the gradients by differentiating them."""
    s = prepare(case, seed)
    with torch.enable_grad():
        return _exact_norm(case, s) if case["op"] == "norm" else _exact_route(case, s)


def _exact_norm(case, s):
    w = s["weight"].double().requires_grad_(case["train"])
    b = None if s["bias"] is None else s["bias"].double().requires_grad_(case["train"])
    total = None if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
    h = (s["x"] if total is None else total).double().requires_grad_(case["train"])
    var, mean = torch.var_mean(h, dim=1, keepdim=True, unbiased=False)
    out = (h - mean) * torch.rsqrt(var + s["eps"]) * w
    if b is not None:
        out = out + b
    found = {"out": out.detach(), "sum": None if total is None else total.double()}
    if case["train"]:
        leaves = [h, w] + ([] if b is None else [b])
        grads = torch.autograd.grad(out, leaves, s["grad_out"].double())
        found["grad"] = grads[0] if s["grad_sum"] is None else grads[0] + s["grad_sum"].double()
        found["grad_weight"] = grads[1]
        found["grad_bias"] = None if b is None else grads[2]
    return found


def _exact_route(case, s):
    z = s["logits"].double()
    n, e = z.shape
    off = z == -math.inf
    x = torch.where(off, 0.0, z).requires_grad_(case["train"] != "no")
    if case["scoring"] == "softmax":
        shifted = torch.where(off, -1e9, x)
        score = torch.where(off, 0.0, torch.softmax(shifted, dim=1))
    else:
        score = torch.where(off, 0.0, torch.sigmoid(x))
    direct = s["balance"] is None and not (case["groups"] > 1 and case["group_score"] == "top2")
    by = z if direct else score.detach() + (0.0 if s["balance"] is None else s["balance"].double())
    by = by.masked_fill(off, -math.inf)
    if case["groups"] > 1:
        runs = by.view(n, case["groups"], -1)
        best = torch.topk(runs, min(2, runs.size(2)), dim=2).values
        of_run = best[..., 0] if case["group_score"] == "max" else best.clamp(min=-1e3).masked_fill(best == -math.inf, 0.0).sum(2)
        of_run = of_run.masked_fill(best[..., 0] == -math.inf, -math.inf)
        ahead = (of_run.unsqueeze(1) > of_run.unsqueeze(2)) | \
            ((of_run.unsqueeze(1) == of_run.unsqueeze(2)) & torch.ones(case["groups"], case["groups"], dtype=torch.bool,
                                                                      device=z.device).tril(-1))
        by = runs.masked_fill((ahead.sum(2) >= case["kept_groups"]).unsqueeze(2), -math.inf).reshape(n, e)
    order = torch.argsort(by, dim=1, descending=True, stable=True)[:, :case["k"]]
    there = by.gather(1, order) > -math.inf
    chosen = torch.zeros_like(by).scatter_(1, order, there.double())
    w = score * chosen
    if case["renormalise"]:
        w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-300)
    w = case["scale"] * w
    by_place = torch.where(there, w.gather(1, order), 0.0)
    found = {"routing": w.detach(), "indices": None, "weights": by_place.detach()}
    if case["train"] != "no":
        target, q = (w, s["grad"].double()) if case["train"] == "routing" else (by_place, s["grad"].double())
        found["grad"] = torch.autograd.grad(target, x, q)[0]
    return found
