"""The operators around the block-sparse products of a routed layer, in plain form and as a user calls them.

  norm      stk.ops.layer_norm, forward or forward and backward (gradients of the rows, the weight and the bias)
  router    stk.ops.top_experts: the softmax over the experts' scores and its top-k, forward or with the scores' gradient
  experts4  the experts' products with 4-bit weights and group scales on routed tokens: stk.ops.gather_matmul_4bit (token rows in, one
            row per slot out) and stk.ops.matmul_4bit_scatter (slot rows in, weighted token rows out)
  matmul4   the same product without routing, stk.ops.matmul_4bit

`own` chooses between the plain form and the library's operators.  A 4-bit weight of input i and output o is scale[i // group][o] *
(code - 8), or, "affine", scale[i // group][o] * code + offset[i // group][o].
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


def _norm(name, direction, rows, size, dtype="bf16"):
    return {"name": name, "op": "norm", "direction": direction, "rows": rows, "size": size, "dtype": dtype}


def _router(name, direction, tokens, experts, top_k, normalize, dtype="bf16"):
    return {"name": name, "op": "router", "direction": direction, "tokens": tokens, "experts": experts, "top_k": top_k, "normalize": normalize, "dtype": dtype}


def _experts4(name, side, tokens, experts, top_k, inputs, outputs, group=128, affine=False, dtype="bf16"):
    return {"name": name, "op": "experts4", "side": side, "tokens": tokens, "experts": experts, "top_k": top_k, "inputs": inputs, "outputs": outputs,
            "group": group, "affine": affine, "dtype": dtype}


def _matmul4(name, tokens, inputs, outputs, group=128, affine=False, dtype="bf16"):
    return {"name": name, "op": "matmul4", "tokens": tokens, "inputs": inputs, "outputs": outputs, "group": group, "affine": affine, "dtype": dtype}


def listed():
    return [
        # the rows of one decoding step of a serving batch
        _norm("norm_decode", "forward", 64, 1024),
        # a training step in front of the layer of the forward benchmark
        _norm("norm_train", "train", 16384, 1024),
        # full precision, a row length that no vector width divides
        _norm("norm_train_odd", "train", 5003, 1151, dtype="fp32"),
        # long rows, many of them: beyond every cache
        _norm("norm_train_large", "train", 32768, 8192),
        # the router of a decoding step, the chosen experts' weights scaled to one
        _router("router_decode", "forward", 64, 64, 2, True),
        # the router of a large training step, scores in full precision
        _router("router_train", "train", 32768, 64, 2, False, dtype="fp32"),
        # many small experts, several of them per token
        _router("router_many_experts", "train", 16384, 256, 8, True),
        # one decoding step of a serving batch, first product: every expert that is hit has its weights read for a handful of rows
        _experts4("experts4_decode_in", "in", 64, 64, 2, 1024, 4096),
        # the second product of the same step
        _experts4("experts4_decode_out", "out", 64, 64, 2, 4096, 1024),
        # the prompts of a serving batch through the first product: 256 rows per expert
        _experts4("experts4_prefill", "in", 16384, 64, 1, 1024, 4096),
        # a single token through a square projection: latency
        _matmul4("matmul4_token", 1, 4096, 4096),
        # a batch that fills no tile, small groups with offsets, an odd number of outputs
        _matmul4("matmul4_batch_odd", 37, 2944, 1151, group=32, affine=True, dtype="fp16"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """An odd size, a multiple of 80 (whole 16-byte pieces, no whole tiles) or a power of two."""
    size, kind = _log_uniform(rng, low, high), rng.random()
    if kind < 0.35:
        return size | 1
    return max(low, size // 80 * 80) if kind < 0.65 else 1 << int(round(math.log2(size)))


def draw(rng):
    op = rng.choice(["norm", "norm", "router", "experts4", "experts4", "matmul4"])
    direction = rng.choice(["forward", "train", "train"])
    if op == "norm":
        size = _size(rng, 16, 16384)
        case = _norm("", direction, min(_log_uniform(rng, 1, 65536), (2 ** 28 - 2 ** 17) // size), size, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if case["dtype"] == "fp32":
            case["rows"] = max(1, case["rows"] // 2)
    elif op == "router":
        experts = _size(rng, 4, 512)
        case = _router("", direction, _log_uniform(rng, 1, 32768), experts, min(experts, rng.choice([1, 2, 2, 4, 8])), rng.random() < 0.5,
                       rng.choice(["bf16", "fp16", "fp32"]))
    else:
        inputs, outputs = _size(rng, 128, 4096), _size(rng, 128, 4096)
        form = (rng.choice([32, 64, 128, 128]), rng.random() < 0.5, rng.choice(["bf16", "bf16", "fp16"]))
        if op == "matmul4":
            case = _matmul4("", _log_uniform(rng, 1, 2048), inputs, outputs, *form)
        else:
            experts = rng.choice([4, 8, 16, 32, 64])
            while experts * inputs * outputs > 2 ** 28:
                experts //= 2
            case = _experts4("", rng.choice(["in", "out"]), _log_uniform(rng, 1, 8192), experts, min(experts, rng.choice([1, 2, 2, 4])), inputs, outputs, *form)
            while case["tokens"] * case["top_k"] * inputs * outputs > 2 ** 36:
                case["tokens"] //= 2
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(shape, std, dtype, gen):
    """N(0, std) values, a slice of rows at a time so that no fp32 copy of a large tensor is made."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    rows = max(1, (1 << 26) // max(1, out[0].numel()))
    for r in range(0, shape[0], rows):
        part = out[r:r + rows]
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen) * std)
    return out


def _prepare_norm(case, gen, dtype):
    rows, size = case["rows"], case["size"]
    # a residual stream: features of different scale and offset
    scale = (torch.randn(size, device="cuda", generator=gen) * 0.5).exp()
    offset = torch.randn(size, device="cuda", generator=gen) * 0.3
    x = _normal((rows, size), 1.0, dtype, gen)
    part = max(1, (1 << 26) // size)
    for r in range(0, rows, part):
        x[r:r + part] = (x[r:r + part].float() * scale + offset).to(dtype)
    s = {"x": x, "weight": (1 + 0.1 * torch.randn(size, device="cuda", generator=gen)).to(dtype),
         "bias": (0.1 * torch.randn(size, device="cuda", generator=gen)).to(dtype)}
    if case["direction"] == "train":
        s["g"] = _normal((rows, size), 1.0, dtype, gen)
        for name in ("x", "weight", "bias"):
            s[name].requires_grad_(True)
    return s


def _prepare_router(case, gen, dtype):
    # experts of unequal popularity, tokens that are sure of their choice to different degrees
    tokens, experts = case["tokens"], case["experts"]
    logits = torch.randn(tokens, experts, device="cuda", generator=gen) * (0.5 + torch.rand(tokens, 1, device="cuda", generator=gen) * 2)
    s = {"logits": (logits + 0.5 * torch.randn(experts, device="cuda", generator=gen)).to(dtype)}
    if case["direction"] == "train":
        s["g"] = torch.randn(tokens, case["top_k"], device="cuda", generator=gen)
        s["logits"].requires_grad_(True)
    return s


def _prepare_weights4(case, experts, gen, dtype):
    inputs, outputs, group = case["inputs"], case["outputs"], case["group"]
    shape = (experts, inputs, outputs) if experts else (inputs, outputs)
    groups = shape[:-2] + ((inputs + group - 1) // group, outputs)
    # codes spread like rounded normal values; the weights' standard deviation is about inputs ** -0.5
    codes = torch.empty(shape, dtype=torch.uint8, device="cuda")
    for part in (codes if experts else [codes]):
        part.copy_((torch.randn(part.shape, device="cuda", generator=gen) * 2.7 + 8).round_().clamp_(0, 15))
    scales = ((0.5 + torch.rand(groups, device="cuda", generator=gen)) * (inputs ** -0.5 / 2.7)).to(dtype)
    offsets = None
    if case["affine"]:
        offsets = (scales.float() * (-8 + 0.5 * torch.randn(groups, device="cuda", generator=gen))).to(dtype)
    s = {"codes": codes, "scales": scales, "offsets": offsets}
    if own:
        import stk_amd as stk
        s["w"] = stk.ops.pack_4bit(codes, scales, group, offsets)   # (laid out once, when a model is loaded)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "norm":
        s.update(_prepare_norm(case, gen, dtype))
    elif case["op"] == "router":
        s.update(_prepare_router(case, gen, dtype))
    elif case["op"] == "matmul4":
        s.update(_prepare_weights4(case, 0, gen, dtype))
        s["x"] = _normal((case["tokens"], case["inputs"]), 1.0, dtype, gen)
    else:
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        s.update(_prepare_weights4(case, experts, gen, dtype))
        s["top"] = torch.rand(tokens, experts, device="cuda", generator=gen).topk(top_k, dim=1).indices.to(torch.int32)
        s["x"] = _normal((tokens if case["side"] == "in" else tokens * top_k, case["inputs"]), 1.0, dtype, gen)
        if case["side"] == "out":
            s["weights"] = torch.rand(tokens, top_k, device="cuda", generator=gen)
        # the routing of the step, which serves both products: the slots by expert and where each expert's end
        order = torch.sort(s["top"].reshape(-1), stable=True)
        s["order"] = order.indices
        s["ends"] = torch.searchsorted(order.values, torch.arange(experts, device="cuda", dtype=torch.int32), right=True).tolist()
        if own:
            import stk_amd as stk
            s["route"] = stk.ops.route(s["top"], experts, 1)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    dtype = s["x"].dtype
    centred = x - x.mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + _EPS)
    xhat = centred * rstd
    y = (xhat * w + b).to(dtype)
    if s["case"]["direction"] == "forward":
        return {"y": y}
    g = s["g"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(dim=1, keepdim=True) - xhat * (gw * xhat).mean(dim=1, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dweight": (g * xhat).sum(dim=0).to(dtype), "dbias": g.sum(dim=0).to(dtype)}


def _plain_router(s):
    case = s["case"]
    logits = s["logits"].detach().float()
    probs = torch.exp(logits - logits.max(dim=1, keepdim=True).values)
    probs = probs / probs.sum(dim=1, keepdim=True)
    experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    weights = torch.gather(probs, 1, experts)
    if case["normalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    out = {"experts": experts.to(torch.int32), "weights": weights}
    if case["direction"] == "train":
        inner = (s["g"] * weights).sum(dim=1, keepdim=True)
        if case["normalize"]:
            grad = torch.zeros_like(probs).scatter(1, experts, weights * (s["g"] - inner))
        else:
            grad = probs * (torch.zeros_like(probs).scatter(1, experts, s["g"]) - inner)
        out["dlogits"] = grad.to(s["logits"].dtype)
    return out


def _plain_weights4(codes, scales, offsets, group):
    rows = torch.arange(codes.shape[0], device=codes.device) // group
    s = scales.float()[rows]
    return codes.float() * s + offsets.float()[rows] if offsets is not None else (codes.float() - 8.0) * s


def _plain_gelu_tanh(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_matmul4(s):
    w = _plain_weights4(s["codes"], s["scales"], s["offsets"], s["case"]["group"])
    return {"y": (s["x"].float() @ w).to(s["x"].dtype)}


def _plain_experts4(s):
    case = s["case"]
    top_k, slots = case["top_k"], case["tokens"] * case["top_k"]
    x = s["x"].float()
    rows = x[s["order"] // top_k] if case["side"] == "in" else x
    y = torch.empty(slots, case["outputs"], device="cuda")
    begin = 0
    for e, end in enumerate(s["ends"]):
        if end > begin:
            w = _plain_weights4(s["codes"][e], s["scales"][e], None if s["offsets"] is None else s["offsets"][e], case["group"])
            y[begin:end] = rows[begin:end] @ w
        begin = end
    if case["side"] == "in":
        return {"h": _plain_gelu_tanh(y).to(s["x"].dtype)}
    by_slot = torch.empty_like(y)
    by_slot[s["order"]] = y
    return {"y": (by_slot.view(case["tokens"], top_k, -1) * s["weights"].unsqueeze(2)).sum(dim=1).to(s["x"].dtype)}


# ---------------------------------------------------------------------------------------------------- one pass
def _own_norm(s):
    import stk_amd as stk
    if s["case"]["direction"] == "forward":
        with torch.no_grad():
            return {"y": stk.ops.layer_norm(s["x"], s["weight"], s["bias"], _EPS)}
    y = stk.ops.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
    dx, dweight, dbias = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["g"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}


def _own_router(s):
    import stk_amd as stk
    case = s["case"]
    if case["direction"] == "forward":
        with torch.no_grad():
            experts, weights = stk.ops.top_experts(s["logits"], case["top_k"], normalize=case["normalize"])
        return {"experts": experts, "weights": weights}
    experts, weights = stk.ops.top_experts(s["logits"], case["top_k"], normalize=case["normalize"])
    dlogits, = torch.autograd.grad(weights, s["logits"], s["g"])
    return {"experts": experts, "weights": weights.detach(), "dlogits": dlogits}


def _own_matmul4(s):
    import stk_amd as stk
    return {"y": stk.ops.matmul_4bit(s["x"], s["w"])}


def _own_experts4(s):
    import stk_amd as stk
    if s["case"]["side"] == "in":
        return {"h": stk.ops.gather_matmul_4bit(s["x"], s["route"], s["w"], "gelu_tanh")}
    return {"y": stk.ops.matmul_4bit_scatter(s["x"], s["route"], s["w"], s["weights"])}


def run(state):
    forms = {"norm": (_plain_norm, _own_norm), "router": (_plain_router, _own_router), "matmul4": (_plain_matmul4, _own_matmul4),
             "experts4": (_plain_experts4, _own_experts4)}
    return forms[state["case"]["op"]][bool(own)](state)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        values = case["rows"] * case["size"]
        if case["direction"] == "forward":      # x, weight, bias in; y out
            return {"bytes": (2 * values + 2 * case["size"]) * e, "flops": 8.0 * values}
        # x and the incoming gradient, weight, bias in; y, three gradients out
        return {"bytes": (4 * values + 4 * case["size"]) * e, "flops": 20.0 * values}
    if case["op"] == "router":
        values, chosen = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        if case["direction"] == "forward":      # scores in; experts and weights out
            return {"bytes": values * e + 8 * chosen, "flops": 4.0 * values}
        return {"bytes": 2 * values * e + 12 * chosen, "flops": 8.0 * values}
    inputs, outputs = case["inputs"], case["outputs"]
    one = inputs * outputs / 2 + (inputs + case["group"] - 1) // case["group"] * outputs * (4 if case["affine"] else 2)
    if case["op"] == "matmul4":
        return {"bytes": one + case["tokens"] * (inputs + outputs) * e, "flops": 2.0 * case["tokens"] * inputs * outputs}
    tokens, slots = case["tokens"], case["tokens"] * case["top_k"]
    hit = case["experts"] * (1.0 - (1.0 - case["top_k"] / case["experts"]) ** tokens)   # experts that get tokens
    rows_in, rows_out = (tokens, slots) if case["side"] == "in" else (slots, tokens)
    return {"bytes": hit * one + (rows_in * inputs + rows_out * outputs) * e, "flops": 2.0 * slots * inputs * outputs}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_norm(s):
    x, weight, bias = (s[name].detach().double() for name in ("x", "weight", "bias"))
    n, train = x.shape[1], s["case"]["direction"] == "train"
    out = {"y": torch.empty_like(x)}
    if train:
        out.update(dx=torch.empty_like(x), dweight=torch.zeros(n, dtype=torch.float64, device="cuda"), dbias=torch.zeros(n, dtype=torch.float64, device="cuda"))
    part = max(1, (1 << 24) // n)
    for r in range(0, x.shape[0], part):
        rows = x[r:r + part]
        var, mean = torch.var_mean(rows, dim=1, correction=0, keepdim=True)
        deviation = (var + _EPS).sqrt()
        z = (rows - mean) / deviation
        out["y"][r:r + part] = torch.addcmul(bias, z, weight)
        if train:
            g = s["g"][r:r + part].double()
            out["dbias"] += g.sum(dim=0)
            out["dweight"] += torch.einsum("rn,rn->n", g, z)
            h = g * weight
            # dz / dx = (1 - 1 1^T / n - z z^T / n) / deviation
            out["dx"][r:r + part] = (h - (h.sum(dim=1, keepdim=True) + z * torch.einsum("rn,rn->r", h, z).unsqueeze(1)) / n) / deviation
    return out


def _exact_router(s):
    case = s["case"]
    logits = s["logits"].detach().double()
    tokens, experts = logits.shape
    log_p = torch.log_softmax(logits, dim=1)
    # rank of every expert: how many are larger, or equal and in front of it
    left, chosen = logits.clone(), []
    places = torch.arange(experts, device="cuda")
    for _ in range(case["top_k"]):
        best = left.amax(dim=1, keepdim=True)
        first = torch.where(left == best, places, experts).amin(dim=1, keepdim=True)
        chosen.append(first)
        left.scatter_(1, first, -math.inf)
    chosen = torch.cat(chosen, dim=1)
    picked = log_p.gather(1, chosen)
    weights = torch.softmax(picked, dim=1) if case["normalize"] else picked.exp()
    out = {"experts": chosen.to(torch.int32), "weights": weights}
    if case["direction"] == "train":
        g = s["g"].double()
        # d weights_j / d logits_i = weights_j (1[i = chosen_j] - q_i), q the softmax over the chosen or over all
        onto = torch.zeros_like(logits).scatter_add_(1, chosen, g * weights)
        q = torch.zeros_like(logits).scatter_(1, chosen, weights) if case["normalize"] else log_p.exp()
        out["dlogits"] = onto - q * (g * weights).sum(dim=1, keepdim=True)
    return out


def _exact_rows4(s, rows, expert):
    """rows @ the weights of one expert (None: the only weights), group by group: sum over g of (rows_g @ codes_g) * scale_g."""
    at = (lambda t: t) if expert is None else (lambda t: t[expert])
    codes, scales, offsets = at(s["codes"]), at(s["scales"]).double(), None if s["offsets"] is None else at(s["offsets"]).double()
    y = torch.zeros(rows.shape[0], codes.shape[1], dtype=torch.float64, device="cuda")
    for g in range(scales.shape[0]):
        part = slice(g * s["case"]["group"], min((g + 1) * s["case"]["group"], codes.shape[0]))
        shift = offsets[g] if offsets is not None else -8.0 * scales[g]
        y += (rows[:, part] @ codes[part].double()) * scales[g] + rows[:, part].sum(dim=1, keepdim=True) * shift
    return y


def _exact_matmul4(s):
    return {"y": _exact_rows4(s, s["x"].double(), None)}


def _exact_experts4(s):
    case = s["case"]
    tokens, top_k = case["tokens"], case["top_k"]
    x, top = s["x"].double(), s["top"].long().cpu()
    slots = sorted(range(tokens * top_k), key=lambda i: int(top.view(-1)[i])) if tokens * top_k <= 4096 else torch.argsort(top.view(-1), stable=True).tolist()
    y = torch.zeros(tokens, case["outputs"], dtype=torch.float64, device="cuda")
    h = torch.empty(len(slots), case["outputs"], dtype=torch.float64, device="cuda")
    position = torch.tensor(slots)
    experts = top.view(-1)[position]
    for e in range(case["experts"]):
        mine = (experts == e).nonzero().view(-1)
        if mine.numel() == 0:
            continue
        slot, mine = position[mine].cuda(), mine.cuda()
        if case["side"] == "in":
            h[mine] = _exact_rows4(s, x[slot // top_k], e)
        else:
            y.index_add_(0, slot // top_k, _exact_rows4(s, x[mine], e) * s["weights"].double().view(-1)[slot].unsqueeze(1))
    if case["side"] == "in":
        return {"h": h * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (h + 0.044715 * h ** 3))}
    return {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "router": _exact_router, "matmul4": _exact_matmul4, "experts4": _exact_experts4}[case["op"]](s)
