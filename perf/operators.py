"""The microscaled 4-bit operators and the routing to experts, as cases whose time is measured.

Three kinds of program call them. A converter, or a tool that looks at a model, quantises tensors to MXFP4 (e2m1 elements, one e8m0
scale per 32 of a row) and takes them back. A server multiplies activations by MXFP4 weights, quantising the activations in the
call: one token per step while it decodes, some tens for a batch, thousands for a prompt. And a server of a mixture of experts
routes tokens to experts and runs the experts' gated feed-forward over MXFP4 weights.

Row lengths and row counts are those of the products measured beside this file (hidden size 5120, feed-forward width 17408, the
H68 block of 4352) and generic ones; experts are a quarter of the hidden size wide.
"""
import math

import torch

own = False   # True: the framework's operators; False: the same mathematics in elementary torch operations

DEVICE = "cuda:0"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _roundtrip(name, M, K, type_, out, acts="normal"):
    return {"name": name, "path": "roundtrip", "M": M, "K": K, "type": type_, "out": out, "acts": acts}


def _product(name, K, N, M, type_, acts="normal"):
    return {"name": name, "path": "product", "K": K, "N": N, "M": M, "type": type_, "acts": acts}


def _route(name, M, E, k, type_, scoring, groups=1, top_groups=1, bias=False, renormalize=True, scale=1.0):
    return {"name": name, "path": "route", "M": M, "E": E, "k": k, "type": type_, "scoring": scoring, "groups": groups,
            "top_groups": top_groups, "bias": bias, "renormalize": renormalize, "scale": scale}


def _experts(name, M, K, F, E, k, absent=0.0, acts="normal", type_="bf16"):
    return {"name": name, "path": "experts", "M": M, "K": K, "F": F, "E": E, "k": k, "type": type_, "absent": absent, "acts": acts}


def listed():
    return [
        # One token's activations to MXFP4 and back: the smallest call of a tool that looks at what quantisation does to them.
        _roundtrip("roundtrip_m1_k5120_bf16", 1, 5120, "bf16", "bf16", acts="outliers"),
        # The activations of a ragged prompt chunk, rows of an odd number of blocks.
        _roundtrip("roundtrip_m1001_k4128_fp16", 1001, 4128, "fp16", "fp32", acts="student_t"),
        # A converter: a feed-forward tensor of fp32 weights.
        _roundtrip("roundtrip_m17408_k5120_fp32", 17408, 5120, "fp32", "fp32", acts="weights"),
        # One product of a decode step, attention-sized.
        _product("product_m1_k5120_n5120_bf16", 5120, 5120, 1, "bf16", acts="outliers"),
        # A short draft checked by the down projection, activations in fp32 as this framework's other products take them.
        _product("product_m3_k17408_n5120_fp32", 17408, 5120, 3, "fp32", acts="relu2"),
        # Some sequences decoded together, an odd number of them and of rows.
        _product("product_m45_k5120_n17401_fp16", 5120, 17401, 45, "fp16", acts="student_t"),
        # A prompt chunk through the feed-forward projection.
        _product("product_m2048_k5120_n17408_bf16", 5120, 17408, 2048, "bf16"),
        # One decoded token's choice among a few experts.
        _route("route_m1_e64_k8_softmax", 1, 64, 8, "fp32", "softmax"),
        # A long prompt's choices among many experts: sigmoid scores, a bias that balances their load, and groups.
        _route("route_m16384_e256_k8_sigmoid_groups", 16384, 256, 8, "fp32", "sigmoid", 8, 4, True, True, 2.5),
        # One decoded token through its experts: their weights are the whole cost.
        _experts("experts_m1_k5120_f1280_e64_k8", 1, 5120, 1280, 64, 8),
        # An odd number of sequences decoded together, experts of an odd number of panels, some of them on another device.
        _experts("experts_m37_k4096_f1376_e60_k4", 37, 4096, 1376, 60, 4, absent=0.25, acts="outliers"),
        # A prompt chunk through all experts: the largest work of such a server's layer.
        _experts("experts_m2048_k5120_f1280_e64_k8", 2048, 5120, 1280, 64, 8),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def _blocks_of(rng, low, high):
    """a row length: a whole number of blocks of 32"""
    return 32 * _log_int(rng, low // 32, high // 32)


def draw(rng):
    kind = rng.random()
    acts = rng.choice(("normal", "outliers", "student_t", "relu2"))
    if kind < 0.2:
        K = _blocks_of(rng, 32, 17408)
        M = _log_int(rng, 1, min(17408, 17408 * 5120 // K))
        c = _roundtrip("", M, K, rng.choice(tuple(TYPES)), rng.choice(("fp32", "bf16")), rng.choice((acts, "weights")))
    elif kind < 0.55:
        K = _blocks_of(rng, 256, 17408)
        N = _log_int(rng, 64, min(17408, 17408 * 5120 // K))
        c = _product("", K, N, _log_int(rng, 1, 2048), rng.choice(tuple(TYPES)), acts)
    elif kind < 0.7:
        groups = rng.choice((1, 1, 2, 4, 8))
        E = groups * _log_int(rng, 8 // groups + 1, 256 // groups)
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, top_groups * (E // groups)))
        c = _route("", _log_int(rng, 1, 16384), E, k, rng.choice(tuple(TYPES)), rng.choice(("softmax", "sigmoid")), groups, top_groups,
                   rng.random() < 0.5, rng.random() < 0.7, rng.choice((1.0, 2.5)))
    else:
        E = rng.randint(4, 64)
        K = _blocks_of(rng, 512, 5120)
        F = _blocks_of(rng, 128, 1280)
        c = _experts("", _log_int(rng, 1, 2048), K, F, E, rng.randint(1, min(8, E)),
                     rng.choice((0.0, 0.0, 0.5)), acts)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _values(kind, M, K, g):
    x = torch.randn((M, K), device=DEVICE, generator=g)
    if kind == "outliers":      # 0.5 % of the channels scaled x20, the same ones for every token
        channels = torch.randperm(K, device=DEVICE, generator=g)[:max(1, round(K * 0.005))]
        x[:, channels] *= 20.0
    elif kind == "student_t":   # Student-t, nu = 4, unit variance
        chi2 = torch.randn((4, M, K), device=DEVICE, generator=g).square().sum(dim=0)
        x = x / (chi2 / 4.0).sqrt() / math.sqrt(2.0)
    elif kind == "relu2":       # behind a squared ReLU: non-negative with a heavy right tail
        x = x.clamp_min(0.0).square()
    elif kind == "weights":     # a trained linear layer's look: rows of different widths
        x = 0.02 * x * (0.5 + torch.rand((M, 1), device=DEVICE, generator=g))
    return x


def _weight(shape, K, g):
    """Codes [*shape, K / 2] and scales [*shape, K / 32] as a model file holds them: elements as of gaussian rows, whose
    deviation is about 2.5 of a block's units, and units around K ** -0.5 / 2.5."""
    p = (torch.arange(256, device=DEVICE, dtype=torch.float32) + 0.5) / 256
    of = 2.5 * math.sqrt(2.0) * torch.erfinv(2 * p - 1)
    nibbles = _code(of).to(torch.int32)                      # 256 equally likely elements
    pair = torch.arange(65536, device=DEVICE, dtype=torch.int32)
    pairs = (nibbles[(pair & 255).long()] | nibbles[(pair >> 8).long()] << 4).to(torch.uint8)
    count = math.prod(shape) * (K // 2)
    which = torch.randint(0, 65536, (count,), device=DEVICE, dtype=torch.int32, generator=g)
    codes = pairs.index_select(0, which).view(*shape, K // 2)
    middle = 127 + round(-0.5 * math.log2(K) - math.log2(2.5))
    scales = torch.randint(middle - 1, middle + 2, (*shape, K // 32), device=DEVICE, dtype=torch.uint8, generator=g)
    return codes, scales


def _inputs(case, seed):
    g = _generator(seed)
    path, M = case["path"], case["M"]
    if path == "roundtrip":
        return {"x": _values(case["acts"], M, case["K"], g).to(TYPES[case["type"]])}
    if path == "product":
        codes, scales = _weight((case["N"],), case["K"], g)
        return {"codes": codes, "scales": scales, "x": _values(case["acts"], M, case["K"], g).to(TYPES[case["type"]])}
    E, k = case["E"], case["k"]
    # a router's logits: experts differ in how often they are asked for
    logits = 1.5 * torch.randn((M, E), device=DEVICE, generator=g) + 0.5 * torch.randn((E,), device=DEVICE, generator=g)
    if path == "route":
        bias = 0.05 * torch.randn((E,), device=DEVICE, generator=g) if case["bias"] else None
        return {"logits": logits.to(TYPES[case["type"]]), "bias": bias}
    top = logits.topk(k, dim=1)
    ids = top.indices.to(torch.int32)
    if case["absent"]:   # experts that another device holds
        ids = torch.where(torch.rand((M, k), device=DEVICE, generator=g) < case["absent"], -1, ids)
    s = {"x": _values(case["acts"], M, case["K"], g).to(TYPES[case["type"]]), "ids": ids, "weights": torch.softmax(top.values, dim=1)}
    s["gate_codes"], s["gate_scales"] = _weight((E, case["F"]), case["K"], g)
    s["up_codes"], s["up_scales"] = _weight((E, case["F"]), case["K"], g)
    s["down_codes"], s["down_scales"] = _weight((E, case["K"]), case["F"], g)
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["path"] in ("product", "experts"):   # what a server keeps: the weights' handles
        import ruquant_amd as rq
        if case["path"] == "product":
            state["weight"] = rq.MXWeight(state["codes"], state["scales"])
        else:
            for name in ("gate", "up", "down"):
                state[name] = rq.MXWeight(state[name + "_codes"], state[name + "_scales"])
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _code(v):
    """e2m1 codes (int32) of values in a block's units: to the nearest, ties to the even code, at most 6"""
    a = v.abs()
    up = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
          + (a > 5.0).int())
    return up + 8 * (v < 0).int()


def _element_table():
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEVICE)
    return torch.cat([t, -t])


def _scale_value(e):
    """2 ** (e - 127) of a scale's byte (int32), NaN for 255"""
    bits = torch.where(e == 0, 0x400000, torch.where(e == 255, 0x7FC00000, e << 23))
    return bits.view(torch.float32)


def _quantised(x):
    """the values that x [.., K] has after quantisation, fp32"""
    v = x.float().unflatten(-1, (-1, 32))
    top = v.abs().amax(dim=-1, keepdim=True).view(torch.int32) >> 23
    e = torch.where(top >= 255, 255, (top - 2).clamp_min(0))
    down = ((254 - e).clamp_min(1) << 23).view(torch.float32)   # 2 ** (127 - e)
    return (_element_table()[_code(v * down)] * _scale_value(e)).flatten(-2)


def _dequantised(codes, scales):
    t = _element_table()
    byte = torch.arange(256, device=DEVICE)
    pairs = torch.stack([t[byte & 15], t[byte >> 4]], dim=1)
    v = pairs.index_select(0, codes.reshape(-1).int()).view(*scales.shape, 32)
    return (v * _scale_value(scales.int())[..., None]).flatten(-2)


def _product_plain(s):
    y = _quantised(s["x"]) @ _dequantised(s["codes"], s["scales"]).t()
    return y.to(s["x"].dtype)


def _route_plain(s):
    case = s["case"]
    x = s["logits"].float()
    if case["scoring"] == "softmax":   # (the sum in 64 bits: its rounding to 32 does not depend on the order)
        e = torch.exp(x - x.amax(dim=1, keepdim=True))
        score = e / e.sum(dim=1, keepdim=True, dtype=torch.float64).float()
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score if s["bias"] is None else score + s["bias"]
    if case["groups"] > 1:
        by = choice.unflatten(1, (case["groups"], -1))
        two = by.sort(dim=2, descending=True).values
        worth = two[:, :, 0] + two[:, :, 1] if two.shape[2] > 1 else two[:, :, 0]
        best = worth.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros_like(worth, dtype=torch.bool).scatter(1, best, True)
        choice = torch.where(kept[:, :, None], by, -math.inf).flatten(1)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]]
    w = score.gather(1, ids)
    if case["renormalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    return ids.to(torch.int32), w * case["scale"]


def _experts_plain(s):
    x, ids, w = s["x"], s["ids"], s["weights"]
    E = s["gate_codes"].shape[0]
    M, k = ids.shape
    here = (ids >= 0) & (ids < E)
    expert = torch.where(here, ids, 0).flatten().long()
    token = torch.arange(M, device=DEVICE).repeat_interleave(k)
    a = _quantised(x)
    if M * k <= E:   # few slots: the weights of each slot's expert
        matrices = [(s[n + "_codes"][expert], s[n + "_scales"][expert]) for n in ("gate", "up", "down")]
        rows = a[token][:, None, :]
        place = (torch.arange(M * k, device=DEVICE), torch.zeros(M * k, dtype=torch.int64, device=DEVICE))
    else:            # many: each expert's tokens side by side
        matrices = [(s[n + "_codes"], s[n + "_scales"]) for n in ("gate", "up", "down")]
        of = torch.nn.functional.one_hot(expert, E).int() * here.flatten()[:, None].int()
        before = of.cumsum(dim=0, dtype=torch.int32)
        place = (expert, (before.gather(1, expert[:, None])[:, 0] - 1).clamp_min(0).long())
        rows = torch.zeros((E, max(1, int(before[-1].max())), x.shape[1]), device=DEVICE)
        at = here.flatten().nonzero()[:, 0]
        rows[place[0][at], place[1][at]] = a[token[at]]
    gate, up, down = (_dequantised(*m) for m in matrices)
    g = torch.bmm(rows, gate.transpose(1, 2).contiguous())
    u = torch.bmm(rows, up.transpose(1, 2).contiguous())
    h = _quantised(g / (1.0 + torch.exp(-g)) * u)
    y = torch.bmm(h, down.transpose(1, 2).contiguous())[place].view(M, k, -1)
    return torch.where(here[:, :, None], y * w[:, :, None], 0.0).sum(dim=1).to(x.dtype)


def run(state):
    case = state["case"]
    path = case["path"]
    if not own:
        if path == "roundtrip":
            return _quantised(state["x"]).to(TYPES[case["out"]])
        return {"product": _product_plain, "route": _route_plain, "experts": _experts_plain}[path](state)
    import ruquant_amd as rq
    if path == "roundtrip":
        codes, scales = rq.mx_quantize(state["x"])
        return rq.mx_dequantize(codes, scales, dtype=TYPES[case["out"]])
    if path == "product":
        return rq.mx_mul_mat(state["weight"], state["x"])
    if path == "route":
        return rq.route(state["logits"], case["k"], scoring=case["scoring"], bias=state["bias"], groups=case["groups"],
                        top_groups=case["top_groups"], renormalize=case["renormalize"], scale=case["scale"])
    return rq.expert_ffn(state["gate"], state["up"], state["down"], state["x"], state["ids"], state["weights"])


def work(case):
    path, M = case["path"], case["M"]
    if path == "route":
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": M * case["E"] * size + (4 * case["E"] if case["bias"] else 0) + 8 * M * case["k"], "flops": 4 * M * case["E"]}
    K = case["K"]
    size = 4 if case["type"] == "fp32" else 2
    if path == "roundtrip":   # (the codes and scales in between are written and read once, by two calls)
        return {"bytes": M * K * (size + (4 if case["out"] == "fp32" else 2)) + 2 * M * (K // 2 + K // 32), "flops": 4 * M * K}
    if path == "product":
        N = case["N"]
        return {"bytes": N * (K // 2 + K // 32) + size * M * (K + N), "flops": 2 * M * N * K}
    E, k, F = case["E"], case["k"], case["F"]
    share = 1.0 - case["absent"]
    asked = E * (1.0 - (1.0 - share * k / E) ** M)   # experts that some token asks for, were all asked for equally often
    return {"bytes": int(asked * 3 * F * (K // 2 + K // 32)) + 2 * size * M * K + 8 * M * k, "flops": int(6 * share * M * k * F * K)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _rounded64(x):
    """x [.., K] in 64 bits -> the nearest MXFP4 values: a block's unit is 2 ** (floor(log2 max) - 2), at least 2 ** -127"""
    v = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    largest = v.abs().max(dim=-1, keepdim=True).values
    power = torch.frexp(largest).exponent - 3                       # (frexp: largest = m * 2 ** p with m in [0.5, 1))
    power = torch.where(largest > 0, power, -127).clamp_min(-127)
    unit = torch.ldexp(torch.ones_like(largest), power)
    v = v / unit
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = (torch.round(a / step) * step).clamp_max(6.0)               # (torch rounds half to even)
    return (torch.sign(v) * q * unit).reshape(x.shape)


def _weight64(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    magnitude, power = c & 1, (c >> 1) & 3
    a = torch.where(power == 0, 0.5 * magnitude.double(), (1.0 + 0.5 * magnitude.double()) * torch.exp2(power.double() - 1.0))
    a = torch.where(c >= 8, -a, a)
    return a * torch.exp2(scales.double() - 127.0).repeat_interleave(32, dim=-1)


def exact(case, seed):
    s = _inputs(case, seed)
    path = case["path"]
    if path == "roundtrip":
        return _rounded64(s["x"])
    if path == "product":
        return torch.matmul(_rounded64(s["x"]), _weight64(s["codes"], s["scales"]).T.contiguous())
    if path == "route":
        x = s["logits"].double()
        score = torch.softmax(x, dim=1) if case["scoring"] == "softmax" else torch.sigmoid(x)
        choice = score if s["bias"] is None else score + s["bias"].double()
        if case["groups"] > 1:
            size = case["E"] // case["groups"]
            worth = choice.reshape(-1, case["groups"], size).topk(min(2, size), dim=2).values.sum(dim=2)
            order = torch.argsort(-worth, dim=1, stable=True)
            rank = torch.argsort(order, dim=1)
            choice = choice.masked_fill((rank >= case["top_groups"]).repeat_interleave(size, dim=1), -math.inf)
        ids = torch.argsort(-choice, dim=1, stable=True)[:, :case["k"]]
        w = torch.take_along_dim(score, ids, dim=1)
        return None, case["scale"] * (w / w.sum(dim=1, keepdim=True) if case["renormalize"] else w)
    x, y = _rounded64(s["x"]), torch.zeros(s["x"].shape, dtype=torch.float64, device=DEVICE)
    for e in range(case["E"]):
        t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not len(t):
            continue
        gate, up, down = (_weight64(s[n + "_codes"][e], s[n + "_scales"][e]).T.contiguous() for n in ("gate", "up", "down"))
        g = torch.matmul(x[t], gate)
        h = _rounded64(g * torch.sigmoid(g) * torch.matmul(x[t], up))
        y.index_add_(0, t, s["weights"][t, j].double()[:, None] * torch.matmul(h, down))
    return y
