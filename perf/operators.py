"""Workloads of the dense projection, the expert router and the mixture-of-experts layer.

Each case is one operator at one size.  ``run`` computes it either with the package's prepared
operators (``own``) or in its plain form: elementary torch operations in 32 bits (the router's
logits and scores in 64, since a choice between neighbouring experts must not depend on the
order of a sum), rounded once at the end.  ``exact`` is the definition in 64 bits.

  linear   y = act(x W^T + b) + r
  route    p = softmax(x W^T) or sigmoid(x W^T); ids = the k experts of the largest p (+ c, a
           bias of the choice only), ties to the lower index; w = p[ids] (/ their sum) * scale;
           a token whose mask is false gets ids -1 and weights 0
  moe      y_t = r_t + sum_j w_tj F_{ids_tj}(x_t), F_e(x) = act(x W1_e^T) W2_e^T; for 'swiglu'
           W1_e = [gate; up] and act = silu(gate) * up
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One generated token through a square projection back into the residual stream.
        {"name": "linear_1x4096x4096", "op": "linear", "m": 1, "k": 4096, "n": 4096, "dtype": "bf16",
         "act": "none", "bias": False, "residual": True, "x_view": "plain"},
        # A decode batch through the up projection of a 4096-wide model, bias and GELU fused.
        {"name": "linear_16x4096x16384", "op": "linear", "m": 16, "k": 4096, "n": 16384, "dtype": "bf16",
         "act": "gelu", "bias": True, "residual": False, "x_view": "plain"},
        # A small model's down projection over 4 x 128 tokens.
        {"name": "linear_512x2048x512", "op": "linear", "m": 512, "k": 2048, "n": 512, "dtype": "fp16",
         "act": "none", "bias": True, "residual": True, "x_view": "plain"},
        # Odd sizes and a transposed input view, as in the strided feed-forward workload.
        {"name": "linear_6993x100x1000", "op": "linear", "m": 6993, "k": 100, "n": 1000, "dtype": "fp16",
         "act": "silu", "bias": True, "residual": True, "x_view": "transposed"},
        # A prompt batch of 8 x 2048 tokens through a square projection with its residual.
        {"name": "linear_16384x4096x4096", "op": "linear", "m": 16384, "k": 4096, "n": 4096, "dtype": "bf16",
         "act": "none", "bias": True, "residual": True, "x_view": "plain"},
        # One token choosing 6 of 64 experts.
        {"name": "route_1x2048_6of64", "op": "route", "m": 1, "k": 2048, "experts": 64, "top": 6, "dtype": "bf16",
         "scoring": "softmax", "choice_bias": False, "renorm": True, "masked": False},
        # A prompt's tokens choosing 8 of 256 by sigmoid scores and a balancing bias, some of them padding.
        {"name": "route_1000x4096_8of256", "op": "route", "m": 1000, "k": 4096, "experts": 256, "top": 8,
         "dtype": "bf16", "scoring": "sigmoid", "choice_bias": True, "renorm": True, "masked": True},
        # One generated token, many small experts.
        {"name": "moe_1x2048_6of64", "op": "moe", "m": 1, "k": 2048, "h": 1024, "n": 2048, "experts": 64, "top": 6,
         "dtype": "bf16", "act": "swiglu", "scoring": "softmax", "choice_bias": False, "renorm": True,
         "residual": True, "masked": False},
        # A decode batch of 16, medium experts.
        {"name": "moe_16x4096_4of32", "op": "moe", "m": 16, "k": 4096, "h": 2048, "n": 4096, "experts": 32, "top": 4,
         "dtype": "bf16", "act": "swiglu", "scoring": "softmax", "choice_bias": False, "renorm": True,
         "residual": True, "masked": False},
        # A padded decode batch of 64 over many small experts, sigmoid scores with a balancing bias.
        {"name": "moe_64x2048_6of64", "op": "moe", "m": 64, "k": 2048, "h": 1024, "n": 2048, "experts": 64, "top": 6,
         "dtype": "bf16", "act": "swiglu", "scoring": "sigmoid", "choice_bias": True, "renorm": True,
         "residual": True, "masked": True},
        # Odd sizes, plain GELU experts, fp16, another output width.
        {"name": "moe_7x500_3of10", "op": "moe", "m": 7, "k": 500, "h": 700, "n": 330, "experts": 10, "top": 3,
         "dtype": "fp16", "act": "gelu", "scoring": "softmax", "choice_bias": False, "renorm": False,
         "residual": False, "masked": False},
        # The most tokens of one call over few large experts.
        {"name": "moe_256x4096_2of8", "op": "moe", "m": 256, "k": 4096, "h": 4096, "n": 4096, "experts": 8, "top": 2,
         "dtype": "bf16", "act": "silu", "scoring": "softmax", "choice_bias": False, "renorm": True,
         "residual": True, "masked": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "route", "moe", "moe"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "linear":
        k, n = _log_int(rng, 64, 8192), _log_int(rng, 64, 16384)
        if rng.random() < 0.5:
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        m = _log_int(rng, 1, min(16384, 16384 * 4096 * 4096 // (k * n)))
        return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": rng.choice(["none", "none", "gelu", "silu"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.6,
                "x_view": rng.choice(["plain", "plain", "plain", "transposed"])}
    experts = rng.choice([8, 10, 16, 32, 60, 64, 128, 256])
    top = rng.randint(1, min(8, experts))
    scoring, choice = rng.choice(["softmax", "sigmoid"]), rng.random() < 0.4
    if op == "route":
        return {"op": op, "m": _log_int(rng, 1, 1000), "k": rng.choice([512, 1000, 2048, 4096]), "experts": experts,
                "top": top, "dtype": dtype, "scoring": scoring, "choice_bias": choice, "renorm": rng.random() < 0.7,
                "masked": rng.random() < 0.4}
    k = _log_int(rng, 128, 4096)
    h = _log_int(rng, 64, max(64, min(4096, 8 * 4096 * 4096 // (experts * k))))
    if rng.random() < 0.6:
        k, h = -(-k // 64) * 64, -(-h // 64) * 64
    return {"op": op, "m": _log_int(rng, 1, 256), "k": k, "h": h, "n": k if rng.random() < 0.8 else _log_int(rng, 64, k),
            "experts": experts, "top": top, "dtype": dtype, "act": rng.choice(["swiglu", "swiglu", "gelu", "silu"]),
            "scoring": scoring, "choice_bias": choice, "renorm": rng.random() < 0.7, "residual": rng.random() < 0.7,
            "masked": rng.random() < 0.3}


def _w1_rows(case):
    return (2 if case["act"] == "swiglu" else 1) * case["h"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    m, k, op = case["m"], case["k"], case["op"]

    def normal(*shape, scale=1.0, dtype=dt):
        t = torch.empty(shape, dtype=dtype, device="cuda")
        return t.normal_(0.0, scale, generator=g)

    s = {"case": case}
    s["x"] = normal(k, m).t() if case.get("x_view") == "transposed" else normal(m, k)
    s["residual"] = normal(m, case["n"]) if case.get("residual") else None
    if op == "linear":
        s["w"] = normal(case["n"], k, scale=k ** -0.5)
        s["bias"] = normal(case["n"], scale=0.5) if case["bias"] else None
    else:
        e = case["experts"]
        s["wr"] = normal(e, k, scale=k ** -0.5)
        s["choice_bias"] = normal(e, scale=0.05, dtype=torch.float32) if case["choice_bias"] else None
        s["mask"] = torch.rand(m, device="cuda", generator=g) > 0.2 if case["masked"] else None
        if op == "moe":
            s["w1"] = normal(e, _w1_rows(case), k, scale=k ** -0.5)
            s["w2"] = normal(e, case["n"], case["h"], scale=case["h"] ** -0.5)
    if own:
        from ffn_optim_b200 import prepare_linear, prepare_moe_ffn, prepare_router

        routing = {} if op == "linear" else dict(top_k=case["top"], scoring=case["scoring"], renormalize=case["renorm"],
                                                 choice_bias=s["choice_bias"], mask=s["mask"])
        if op == "linear":
            s["op"] = prepare_linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"], activation=case["act"],
                                     gelu="erf")
        elif op == "route":
            s["op"] = prepare_router(s["x"], s["wr"], **routing)
        else:
            s["op"] = prepare_moe_ffn(s["x"], s["wr"], s["w1"], s["w2"], activation=case["act"], gelu="erf",
                                      residual=s["residual"], **routing)
    return s


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "swiglu":
        gate, up = z.chunk(2, dim=-1)
        return gate / (1.0 + torch.exp(-gate)) * up
    return z


def _plain_linear(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    z = _act(z, s["case"]["act"])
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(s["x"].dtype)


def _plain_route(s):
    case = s["case"]
    logits = s["x"].double() @ s["wr"].double().t()
    if case["scoring"] == "softmax":
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    key = p if s["choice_bias"] is None else p + s["choice_bias"].double()
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    w = p.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    if s["mask"] is not None:
        ids = torch.where(s["mask"][:, None], ids, -1)
        w = torch.where(s["mask"][:, None], w, 0.0)
    return ids.to(torch.int32), w.float()


def _plain_moe(s):
    case = s["case"]
    x, (m, top, e) = s["x"].float(), (case["m"], case["top"], case["experts"])
    ids, w = _plain_route(s)
    ids = ids.long().clamp(min=0)
    if m * top <= e:  # fewer choices than experts: only the chosen experts' weights are read
        at = ids.reshape(-1)
        z = torch.matmul(s["w1"][at].float(), x.repeat_interleave(top, 0)[:, :, None])[:, :, 0]
        y = torch.matmul(s["w2"][at].float(), _act(z, case["act"])[:, :, None])[:, :, 0]
        y = (y * w.reshape(-1, 1)).reshape(m, top, -1).sum(1)
    else:
        z = torch.matmul(x, s["w1"].float().transpose(1, 2))
        y = torch.matmul(_act(z, case["act"]), s["w2"].float().transpose(1, 2))
        y = (y * torch.zeros(m, e, device=w.device).scatter_add_(1, ids, w).t()[:, :, None]).sum(0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "linear":
            return s["op"].run(s["x"], residual=s["residual"])
        if op == "route":
            return s["op"].run(s["x"], mask=s["mask"])
        return s["op"].run(s["x"], residual=s["residual"], mask=s["mask"])
    return {"linear": _plain_linear, "route": _plain_route, "moe": _plain_moe}[op](s)


def work(case):
    m, k = case["m"], case["k"]
    if case["op"] == "linear":
        n = case["n"]
        values = m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        return {"bytes": 2.0 * values, "flops": 2.0 * m * n * k}
    e, top = case["experts"], case["top"]
    tokens = m * (0.8 if case["masked"] else 1.0)  # a masked token asks for no expert
    route = {"bytes": 2.0 * (tokens * k + e * k) + 8.0 * m * top, "flops": 2.0 * tokens * e * k}
    if case["op"] == "route":
        return route
    h, n = case["h"], case["n"]
    per_expert = _w1_rows(case) * k + n * h
    active = e * (1.0 - (1.0 - top / e) ** tokens)  # experts that at least one token chose, evenly spread choices
    return {"bytes": 2.0 * (active * per_expert + tokens * k + e * k + m * n * (2 if case["residual"] else 1)),
            "flops": 2.0 * tokens * top * per_expert + route["flops"]}


def _exact_act(z, act):
    if act == "swiglu":
        half = z.shape[-1] // 2
        return z[..., :half] * torch.sigmoid(z[..., :half]) * z[..., half:]
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(z) if act == "silu" else z


def _exact_route(s):
    case = s["case"]
    score = torch.einsum("mk,ek->me", s["x"].double(), s["wr"].double())
    score = torch.softmax(score, 1) if case["scoring"] == "softmax" else torch.sigmoid(score)
    key = score.clone()
    if s["choice_bias"] is not None:
        key += s["choice_bias"].double()
    ids, w = [], []
    for _ in range(case["top"]):
        best = key.argmax(1)  # one of the largest; the lowest index among equal ones:
        best = torch.where(key == key.gather(1, best[:, None]), torch.arange(key.shape[1], device=key.device),
                           key.shape[1]).amin(1)
        ids.append(best)
        w.append(score.gather(1, best[:, None])[:, 0])
        key.scatter_(1, best[:, None], -math.inf)
    ids, w = torch.stack(ids, 1), torch.stack(w, 1)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    if s["mask"] is not None:
        ids[~s["mask"]] = -1
        w[~s["mask"]] = 0.0
    return ids.to(torch.int32), w


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    x = s["x"].double()
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    if case["op"] == "linear":
        for lo in range(0, case["m"], 4096):
            z = torch.einsum("mk,nk->mn", x[lo:lo + 4096], s["w"].double())
            if s["bias"] is not None:
                z += s["bias"].double()
            y[lo:lo + 4096] = _exact_act(z, case["act"])
    else:
        ids, w = _exact_route(s)
        for e in range(case["experts"]):
            token, place = torch.nonzero(ids == e, as_tuple=True)
            if token.numel():
                hidden = _exact_act(torch.einsum("mk,hk->mh", x[token], s["w1"][e].double()), case["act"])
                y[token] += torch.einsum("mh,nh->mn", hidden, s["w2"][e].double()) * w[token, place][:, None]
    return y if s["residual"] is None else y + s["residual"].double()
