"""More operators around the block-sparse products of a routed layer, in plain form and as a user calls them.

  router   stk.ops.group_top_experts: the choice among groups of experts, from softmax or sigmoid scores with a bias for balance, forward or with
           the scores' gradient
  matmul8  stk.ops.matmul_8bit: rows times 8-bit floating-point weights that have a scale for every block of 128 x 128
  experts8 the experts' products with such weights on routed tokens: stk.ops.gather_matmul_8bit (token rows in, one row per slot out)
           and stk.ops.matmul_8bit_scatter (slot rows in, weighted token rows out)
  linear8  stk.ops.linear_8bit: the product of a training step with weights that are trained, forward and both gradients, one matrix or the
           experts' on the padded layout of a routing

`own` chooses between the plain form and the library's operators.  8-bit values are e4m3 (4 bits of exponent, 3 of mantissa, at most 448).  What a
product multiplies is quantised within the call with scales that are powers of two, the smallest 2^e (e >= -126) with max |x| <= 448 2^e: rows
for every 128 inputs; trained weights for every block of 128 x 128; for the gradient of the weights, rows and incoming gradients for
every 128 rows of a column.  Stored weights have scales of that kind ("e8m0") or any ("float").
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 128


def _router(name, direction, tokens, experts, groups, top_groups, top_k, scoring, bias, group_best, normalize, scale, dtype):
    return {"name": name, "op": "router", "direction": direction, "tokens": tokens, "experts": experts, "groups": groups, "top_groups": top_groups,
            "top_k": top_k, "scoring": scoring, "bias": bias, "group_best": group_best, "normalize": normalize, "scale": scale, "dtype": dtype}


def _matmul8(name, tokens, inputs, outputs, scales="e8m0", dtype="bf16"):
    return {"name": name, "op": "matmul8", "tokens": tokens, "inputs": inputs, "outputs": outputs, "scales": scales, "dtype": dtype}


def _experts8(name, side, tokens, experts, top_k, inputs, outputs, scales="e8m0", dtype="bf16"):
    return {"name": name, "op": "experts8", "side": side, "tokens": tokens, "experts": experts, "top_k": top_k, "inputs": inputs, "outputs": outputs,
            "scales": scales, "dtype": dtype}


def _linear8(name, tokens, experts, top_k, inputs, outputs, dtype="bf16"):
    """experts 0: one matrix."""
    return {"name": name, "op": "linear8", "tokens": tokens, "experts": experts, "top_k": top_k, "inputs": inputs, "outputs": outputs, "dtype": dtype}


def listed():
    return [
        # the router of a decoding step: many small experts in groups, balanced by a bias
        _router("router_decode", "forward", 64, 256, 8, 4, 8, "sigmoid", True, 2, True, 2.5, "fp32"),
        # the same router in a large training step
        _router("router_train", "train", 16384, 256, 8, 4, 8, "sigmoid", True, 2, True, 2.5, "fp32"),
        # softmax scores without a bias, groups of a size that no power of two is, an odd number of tokens
        _router("router_softmax_odd", "train", 20005, 160, 8, 3, 6, "softmax", False, 1, False, 16.0, "bf16"),
        # a single token through a square projection: latency
        _matmul8("matmul8_token", 1, 4096, 4096),
        # a batch that fills no tile, an odd number of outputs, weights from elsewhere with scales of any value
        _matmul8("matmul8_batch_odd", 37, 2944, 1151, scales="float", dtype="fp16"),
        # the prompts of a serving batch through a square projection
        _matmul8("matmul8_prompts", 8192, 4096, 4096, scales="float"),
        # one decoding step of a serving batch, first product: every expert that is hit has its weights read for a handful of rows
        _experts8("experts8_decode_in", "in", 64, 64, 2, 1024, 4096),
        # the second product of the same step
        _experts8("experts8_decode_out", "out", 64, 64, 2, 4096, 1024),
        # the prompts of a serving batch through the first product: 256 rows per expert
        _experts8("experts8_prefill", "in", 16384, 64, 1, 1024, 4096),
        # a training step of a large dense projection
        _linear8("linear8_train", 16384, 0, 1, 4096, 4096),
        # sizes that fill no block
        _linear8("linear8_odd", 2501, 0, 1, 1151, 2944, dtype="fp16"),
        # the experts' first product in a training step of the layer of the forward benchmark
        _linear8("linear8_experts", 16384, 64, 1, 1024, 4096),
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
    op = rng.choice(["router", "router", "matmul8", "experts8", "experts8", "linear8", "linear8"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "router":
        groups = rng.choice([1, 2, 4, 6, 8, 16])
        each = rng.randint(max(2, 8 // groups), min(64, 512 // groups))
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(12, top_groups * each))
        case = _router("", rng.choice(["forward", "train", "train"]), _log_uniform(rng, 1, 32768), groups * each, groups, top_groups, top_k,
                       rng.choice(["softmax", "sigmoid"]), rng.random() < 0.6, rng.choice([1, 2]), rng.random() < 0.6, rng.choice([1.0, 2.5, 16.0]),
                       rng.choice(["bf16", "fp32", "fp32"]))
    elif op == "matmul8":
        case = _matmul8("", _log_uniform(rng, 1, 8192), _size(rng, 128, 4096), _size(rng, 128, 4096), rng.choice(["e8m0", "float"]), dtype)
    elif op == "experts8":
        inputs, outputs, experts = _size(rng, 128, 4096), _size(rng, 128, 4096), rng.choice([4, 8, 16, 32, 64])
        while experts * inputs * outputs > 2 ** 28:
            experts //= 2
        case = _experts8("", rng.choice(["in", "out"]), _log_uniform(rng, 1, 8192), experts, min(experts, rng.choice([1, 2, 2, 4])), inputs, outputs,
                         rng.choice(["e8m0", "float"]), dtype)
        while case["tokens"] * case["top_k"] * inputs * outputs > 2 ** 36:
            case["tokens"] //= 2
    else:
        inputs, outputs, experts = _size(rng, 128, 4096), _size(rng, 128, 4096), rng.choice([0, 0, 4, 8, 16])
        while experts * inputs * outputs > 2 ** 27:
            experts //= 2
        case = _linear8("", _log_uniform(rng, 1, 16384), experts, 1 if experts < 2 else rng.choice([1, 2]), inputs, outputs, dtype)
        while case["tokens"] * case["top_k"] * inputs * outputs > 2 ** 37:
            case["tokens"] //= 2
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- the 8-bit format
def _to_blocks(x, rows, cols):
    """x padded with zeros to whole blocks, as [row blocks, rows, column blocks, cols]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // cols, cols)


def _power(exponent):
    """2^exponent in fp32, exponents of normal numbers."""
    return ((exponent + 127) << 23).to(torch.int32).view(torch.float32)


def _quantised(x, rows, cols):
    """(codes, scales [row blocks, column blocks]): e4m3 values and the power of two of every rows x cols block of x."""
    blocks = _to_blocks(x.float(), rows, cols)
    most = blocks.abs().amax(dim=(1, 3))
    mantissa, exponent = torch.frexp(most)                     # most = mantissa 2^exponent, mantissa in [0.5, 1); 448 = 0.875 2^9
    exponent = (exponent - 9 + (mantissa > 0.875)).clamp(min=-126)
    exponent = torch.where(most == 0, -126, exponent)
    codes = (blocks * _power(-exponent)[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.view(blocks.shape[0] * rows, -1)[:x.shape[0], :x.shape[1]].contiguous()
    return codes, _power(exponent)


def _values(codes, scales, rows, cols):
    """What codes and scales stand for, fp32."""
    blocks = _to_blocks(codes.float(), rows, cols) * scales.float()[:, None, :, None]
    return blocks.view(blocks.shape[0] * rows, -1)[:codes.shape[0], :codes.shape[1]]


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(shape, std, dtype, gen):
    """N(0, std) values, a slice of rows at a time so that no fp32 copy of a large tensor is made."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    rows = max(1, (1 << 26) // max(1, out[0].numel()))
    for r in range(0, shape[0], rows):
        part = out[r:r + rows]
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen) * std)
    return out


def _activations(rows, size, dtype, gen):
    """Rows as a norm leaves them: features of different size, a few of them far larger than the others."""
    feature = (torch.randn(size, device="cuda", generator=gen) * 0.5).exp()
    feature[torch.randint(0, size, (max(1, size // 256),), device="cuda", generator=gen)] *= 20
    out = _normal((rows, size), 1.0, dtype, gen)
    part = max(1, (1 << 26) // size)
    for r in range(0, rows, part):
        out[r:r + part] = (out[r:r + part].float() * feature).to(dtype)
    return out


def _prepare_router(case, gen, dtype):
    # experts of unequal popularity, tokens that are sure of their choice to different degrees
    tokens, experts = case["tokens"], case["experts"]
    scores = torch.randn(tokens, experts, device="cuda", generator=gen) * (0.5 + torch.rand(tokens, 1, device="cuda", generator=gen))
    popularity = 0.5 * torch.randn(experts, device="cuda", generator=gen)
    s = {"scores": (scores + popularity).to(dtype), "bias": None}
    if case["bias"]:
        # what balancing has made of it: against the popularity, in steps
        size = 0.2 if case["scoring"] == "sigmoid" else 0.5 / experts
        s["bias"] = torch.round(-popularity * size * 1000 + torch.randn(experts, device="cuda", generator=gen)) / 1000
    if case["direction"] == "train":
        s["g"] = torch.randn(tokens, case["top_k"], device="cuda", generator=gen)
        s["scores"].requires_grad_(True)
    return s


def _prepare_weights8(case, experts, gen):
    inputs, outputs = case["inputs"], case["outputs"]
    count = max(1, experts)
    blocks = ((inputs + _BLOCK - 1) // _BLOCK, (outputs + _BLOCK - 1) // _BLOCK)
    codes = torch.empty((count, inputs, outputs), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((count, *blocks), device="cuda")
    for e in range(count):
        w = torch.randn(inputs, outputs, device="cuda", generator=gen) * inputs ** -0.5
        if case["scales"] == "float":   # codes of weights that were divided by scales of any value
            scales[e] = (0.7 + 0.6 * torch.rand(blocks, device="cuda", generator=gen)) * inputs ** -0.5 / 80
            wide = scales[e].repeat_interleave(_BLOCK, 0).repeat_interleave(_BLOCK, 1)[:inputs, :outputs]
            codes[e] = (w / wide).clamp(-448, 448).to(torch.float8_e4m3fn)
        else:
            codes[e], scales[e] = _quantised(w, _BLOCK, _BLOCK)
    if not experts:
        codes, scales = codes[0], scales[0]
    s = {"codes": codes, "scales": scales}
    if own:
        import stk_amd as stk
        s["w"] = stk.ops.pack_8bit(codes, scales.to(torch.float8_e8m0fnu) if case["scales"] == "e8m0" else scales)   # (once, when a model is loaded)
    return s


def _prepare_routing(case, gen, blocking, padded_rows=None):
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    top = torch.rand(tokens, experts, device="cuda", generator=gen).topk(top_k, dim=1).indices.to(torch.int32)
    order = torch.sort(top.reshape(-1), stable=True)
    ends = torch.searchsorted(order.values, torch.arange(experts, device="cuda", dtype=torch.int32), right=True).tolist()
    s = {"top": top, "order": order.indices, "ends": ends}
    if own:
        import stk_amd as stk
        s["route"] = stk.ops.route(top, experts, blocking, padded_rows)
    return s


def _prepare_linear8(case, gen, dtype):
    inputs, outputs, experts = case["inputs"], case["outputs"], case["experts"]
    s = {"w": _normal((max(1, experts), inputs, outputs), inputs ** -0.5, dtype, gen)}
    s["x"], s["g"] = _activations(case["tokens"] * case["top_k"], inputs, dtype, gen), _normal((case["tokens"] * case["top_k"], outputs), 1e-4, dtype, gen)
    s["parts"] = [(0, case["tokens"])]
    if experts:
        # the rows in the padded layout of a routing: every expert's rows, then zeros up to a multiple of 128; behind the last expert zeros, as many
        # as any routing of so many tokens may need
        rows = (case["tokens"] * case["top_k"] + experts * (_BLOCK - 1)) // _BLOCK * _BLOCK
        s.update(_prepare_routing(case, gen, _BLOCK, rows))
        s["parts"], place, at, begin = [], [], 0, 0
        for end in s["ends"]:
            place.append(torch.arange(at, at + end - begin))
            s["parts"].append((at, at + (end - begin + _BLOCK - 1) // _BLOCK * _BLOCK))
            at, begin = s["parts"][-1][1], end
        place = torch.cat(place).to("cuda")
        for name in ("x", "g"):
            s[name] = torch.zeros(rows, s[name].shape[1], dtype=dtype, device="cuda").index_copy_(0, place, s[name])
    else:
        s["w"] = s["w"][0]
    s["x"].requires_grad_(True)
    s["w"].requires_grad_(True)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "router":
        s.update(_prepare_router(case, gen, dtype))
    elif case["op"] == "linear8":
        s.update(_prepare_linear8(case, gen, dtype))
    elif case["op"] == "matmul8":
        s.update(_prepare_weights8(case, 0, gen))
        s["x"] = _activations(case["tokens"], case["inputs"], dtype, gen)
    else:
        s.update(_prepare_weights8(case, case["experts"], gen))
        s.update(_prepare_routing(case, gen, 1))
        s["x"] = _activations(case["tokens"] * (1 if case["side"] == "in" else case["top_k"]), case["inputs"], dtype, gen)
        if case["side"] == "out":
            s["weights"] = torch.rand(case["tokens"], case["top_k"], device="cuda", generator=gen)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_router(s):
    case = s["case"]
    scores = s["scores"].detach().double()   # (in 64 bits: two experts may be chosen on a difference that 32 lose)
    tokens, experts = scores.shape
    if case["scoring"] == "softmax":
        p = torch.exp(scores - scores.max(dim=1, keepdim=True).values)
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-scores))
    choice = p if s["bias"] is None else p + s["bias"].double()
    groups = case["groups"]
    best = torch.sort(choice.view(tokens, groups, -1), dim=2, descending=True).values[:, :, :case["group_best"]].sum(dim=2)
    kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
    out_of = torch.ones_like(best).scatter(1, kept, 0.0).bool().repeat_interleave(experts // groups, 1)
    order = (scores if s["bias"] is None else choice).masked_fill(out_of, -math.inf)
    chosen = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    mine = p.gather(1, chosen)
    total = mine.sum(dim=1, keepdim=True) if case["normalize"] else 1.0
    weights = case["scale"] * mine / total
    out = {"experts": chosen.to(torch.int32), "weights": weights.float()}
    if case["direction"] == "train":
        g = s["g"].double() * case["scale"]
        if case["normalize"]:
            g = (g - (g * mine).sum(dim=1, keepdim=True) / total) / total
        onto = torch.zeros_like(p).scatter(1, chosen, g)
        if case["scoring"] == "softmax":
            grad = p * (onto - (onto * p).sum(dim=1, keepdim=True))
        else:
            grad = onto * p * (1.0 - p)
        out["dscores"] = grad.to(s["scores"].dtype)
    return out


def _plain_rows(x):
    codes, scales = _quantised(x, 1, _BLOCK)
    return _values(codes, scales, 1, _BLOCK)


def _plain_columns(x):
    codes, scales = _quantised(x, _BLOCK, 1)
    return _values(codes, scales, _BLOCK, 1)


def _plain_gelu_tanh(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_matmul8(s):
    return {"y": (_plain_rows(s["x"]) @ _values(s["codes"], s["scales"], _BLOCK, _BLOCK)).to(s["x"].dtype)}


def _plain_experts8(s):
    case = s["case"]
    top_k, slots = case["top_k"], case["tokens"] * case["top_k"]
    x = _plain_rows(s["x"])
    rows = x[s["order"] // top_k] if case["side"] == "in" else x
    y = torch.empty(slots, case["outputs"], device="cuda")
    begin = 0
    for e, end in enumerate(s["ends"]):
        if end > begin:
            y[begin:end] = rows[begin:end] @ _values(s["codes"][e], s["scales"][e], _BLOCK, _BLOCK)
        begin = end
    if case["side"] == "in":
        return {"h": _plain_gelu_tanh(y).to(s["x"].dtype)}
    by_slot = torch.empty_like(y)
    by_slot[s["order"]] = y
    return {"y": (by_slot.view(case["tokens"], top_k, -1) * s["weights"].unsqueeze(2)).sum(dim=1).to(s["x"].dtype)}


def _plain_linear8(s):
    x, g, w = s["x"].detach(), s["g"], s["w"].detach()
    w = w if w.dim() == 3 else w.unsqueeze(0)
    y, dx, dw = torch.zeros_like(g), torch.zeros_like(x), torch.empty_like(w)
    for e, (begin, end) in enumerate(s["parts"]):
        codes, scales = _quantised(w[e], _BLOCK, _BLOCK)
        we = _values(codes, scales, _BLOCK, _BLOCK)
        y[begin:end] = (_plain_rows(x[begin:end]) @ we).to(y.dtype)
        dx[begin:end] = (_plain_rows(g[begin:end]) @ we.t()).to(dx.dtype)
        dw[e] = (_plain_columns(x[begin:end]).t() @ _plain_columns(g[begin:end])).to(dw.dtype) if end > begin else 0
    return {"y": y, "dx": dx, "dw": dw.view(s["w"].shape)}


# ---------------------------------------------------------------------------------------------------- one pass
def _own_router(s):
    import stk_amd as stk
    case = s["case"]

    def call():
        return stk.ops.group_top_experts(s["scores"], case["top_k"], groups=case["groups"], top_groups=case["top_groups"], scoring=case["scoring"],
                                         bias=s["bias"], group_best=case["group_best"], normalize=case["normalize"], scale=case["scale"])

    if case["direction"] == "forward":
        with torch.no_grad():
            experts, weights = call()
        return {"experts": experts, "weights": weights}
    experts, weights = call()
    dscores, = torch.autograd.grad(weights, s["scores"], s["g"])
    return {"experts": experts, "weights": weights.detach(), "dscores": dscores}


def _own_matmul8(s):
    import stk_amd as stk
    return {"y": stk.ops.matmul_8bit(s["x"], s["w"])}


def _own_experts8(s):
    import stk_amd as stk
    if s["case"]["side"] == "in":
        return {"h": stk.ops.gather_matmul_8bit(s["x"], s["route"], s["w"], "gelu_tanh")}
    return {"y": stk.ops.matmul_8bit_scatter(s["x"], s["route"], s["w"], s["weights"])}


def _own_linear8(s):
    import stk_amd as stk
    y = stk.ops.linear_8bit(s["x"], s["w"], s.get("route"))
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["g"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def run(state):
    forms = {"router": (_plain_router, _own_router), "matmul8": (_plain_matmul8, _own_matmul8), "experts8": (_plain_experts8, _own_experts8),
             "linear8": (_plain_linear8, _own_linear8)}
    return forms[state["case"]["op"]][bool(own)](state)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "router":
        values, chosen = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        bias = 4 * case["experts"] if case["bias"] else 0
        if case["direction"] == "forward":      # scores in; experts and weights out
            return {"bytes": values * e + bias + 8 * chosen, "flops": 6.0 * values}
        return {"bytes": 2 * values * e + bias + 12 * chosen, "flops": 10.0 * values}
    tokens, inputs, outputs, experts = case["tokens"], case["inputs"], case["outputs"], case.get("experts", 0)
    slots = tokens * case.get("top_k", 1)
    hit = experts * (1.0 - (1.0 - case["top_k"] / experts) ** tokens) if experts else 1.0   # experts that get tokens
    if case["op"] == "linear8":                 # rows, weights, gradient in; result, two gradients out
        return {"bytes": (2 * slots * (inputs + outputs) + (hit + max(1, experts)) * inputs * outputs) * e, "flops": 6.0 * slots * inputs * outputs}
    blocks = ((inputs + _BLOCK - 1) // _BLOCK) * ((outputs + _BLOCK - 1) // _BLOCK)
    one = inputs * outputs + blocks * (4 if case["scales"] == "float" else 1)
    rows_in, rows_out = (slots, tokens) if case.get("side") == "out" else (tokens, slots)
    return {"bytes": hit * one + (rows_in * inputs + rows_out * outputs) * e, "flops": 2.0 * slots * inputs * outputs}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_router(s):
    case = s["case"]
    scores = s["scores"].detach().double()
    tokens, experts = scores.shape
    soft = case["scoring"] == "softmax"
    log_p = torch.log_softmax(scores, dim=1) if soft else torch.nn.functional.logsigmoid(scores)
    value = log_p.exp()
    if s["bias"] is not None:
        value = value + s["bias"].double()
    every = torch.arange(tokens, device="cuda")

    def largest(left, count):
        """Places of the `count` largest of every row, the first of equal ones, one after the other."""
        left, found = left.clone(), []
        places = torch.arange(left.shape[1], device="cuda")
        for _ in range(count):
            found.append(torch.where(left == left.amax(dim=1, keepdim=True), places, left.shape[1]).amin(dim=1))
            left[every, found[-1]] = -math.inf
        return torch.stack(found, dim=1)

    size = experts // case["groups"]
    of_group = torch.stack([value[:, g * size:(g + 1) * size].topk(case["group_best"], dim=1).values.sum(dim=1) for g in range(case["groups"])], dim=1)
    kept = largest(of_group, case["top_groups"])
    inside = torch.zeros(tokens, case["groups"], dtype=torch.bool, device="cuda")
    inside[every.unsqueeze(1), kept] = True
    inside = inside[:, torch.arange(experts, device="cuda") // size]
    chosen = largest(torch.where(inside, scores if s["bias"] is None else value, -math.inf), case["top_k"])
    picked = log_p.gather(1, chosen)
    share = torch.softmax(picked, dim=1) if case["normalize"] else picked.exp()
    out = {"experts": chosen.to(torch.int32), "weights": case["scale"] * share}
    if case["direction"] == "train":
        # through log p: w_j = scale share_j, d share_j / d log p_i = share_j (1[i = j] - share_i) normalised, share_j 1[i = j] otherwise
        g = s["g"].double() * out["weights"]
        if case["normalize"]:
            g = g - share * g.sum(dim=1, keepdim=True)
        if soft:
            out["dscores"] = torch.zeros_like(scores).scatter_add_(1, chosen, g) - log_p.exp() * g.sum(dim=1, keepdim=True)
        else:
            out["dscores"] = torch.zeros_like(scores).scatter_add_(1, chosen, g * torch.special.expit(-scores.gather(1, chosen)))
    return out


def _exact_e4m3(x, axes):
    """x [..., as blocks] rounded to e4m3 with one power of two over `axes`, in 64 bits: a step is 2^(exponent - 3), or 2^-9 below 2^-6."""
    most = x.abs().amax(dim=axes, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(most / 448)).clamp(-126, 200))
    scale = torch.where(most > 448 * scale, scale * 2, scale)              # (a logarithm next to a whole number)
    scale = torch.where((most <= 224 * scale) & (scale > 2.0 ** -126), scale / 2, scale)
    x = x / scale
    step = torch.exp2(torch.frexp(x).exponent.clamp(min=-5).double() - 4)
    return torch.round(x / step) * step * scale


def _exact_rows(x):
    parts = [_exact_e4m3(part, (1,)) for part in x.double().split(_BLOCK, dim=1)]
    return torch.cat(parts, dim=1)


def _exact_columns(x):
    return _exact_rows(x.t()).t()


def _exact_blocks(w):
    return torch.cat([torch.cat([_exact_e4m3(part, (0, 1)) for part in rows.split(_BLOCK, dim=1)], dim=1) for rows in w.double().split(_BLOCK, dim=0)], dim=0)


def _exact_product(s, rows, expert):
    """Quantised rows times stored weights, block by block: sum over blocks of (rows_b @ codes_b) * scale_b."""
    codes, scales = (s["codes"], s["scales"]) if expert is None else (s["codes"][expert], s["scales"][expert])
    wide = scales.double().repeat_interleave(_BLOCK, 1)[:, :codes.shape[1]]
    y = torch.zeros(rows.shape[0], codes.shape[1], dtype=torch.float64, device="cuda")
    for b in range(scales.shape[0]):
        part = slice(b * _BLOCK, min((b + 1) * _BLOCK, codes.shape[0]))
        y += (rows[:, part] @ codes[part].float().double()) * wide[b]
    return y


def _exact_matmul8(s):
    return {"y": _exact_product(s, _exact_rows(s["x"]), None)}


def _exact_experts8(s):
    case = s["case"]
    tokens, top_k = case["tokens"], case["top_k"]
    x, experts = _exact_rows(s["x"]), s["top"].long().view(-1)
    slots = torch.argsort(experts, stable=True)
    mine = experts[slots]
    h = torch.empty(slots.numel(), case["outputs"], dtype=torch.float64, device="cuda")
    y = torch.zeros(tokens, case["outputs"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        at = (mine == e).nonzero().view(-1)
        if at.numel() == 0:
            continue
        if case["side"] == "in":
            h[at] = _exact_product(s, x[slots[at] // top_k], e)
        else:
            y.index_add_(0, slots[at] // top_k, _exact_product(s, x[at], e) * s["weights"].double().view(-1)[slots[at]].unsqueeze(1))
    if case["side"] == "in":
        return {"h": h * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (h + 0.044715 * h ** 3))}
    return {"y": y}


def _exact_linear8(s):
    x, g, w = s["x"].detach(), s["g"], s["w"].detach()
    single = w.dim() == 2
    out = {"y": torch.zeros(g.shape, dtype=torch.float64, device="cuda"), "dx": torch.zeros(x.shape, dtype=torch.float64, device="cuda"),
           "dw": torch.zeros(w.shape, dtype=torch.float64, device="cuda")}
    for e, (begin, end) in enumerate(s["parts"]):
        if begin == end:
            continue
        we, rows = _exact_blocks(w if single else w[e]), slice(begin, end)
        out["y"][rows] = torch.mm(_exact_rows(x[rows]), we)
        out["dx"][rows] = torch.mm(_exact_rows(g[rows]), we.t())
        torch.mm(_exact_columns(x[rows]).t(), _exact_columns(g[rows]), out=out["dw"] if single else out["dw"][e])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"router": _exact_router, "matmul8": _exact_matmul8, "experts8": _exact_experts8, "linear8": _exact_linear8}[case["op"]](s)
