"""The 8-bit integer product and the products grouped by expert, as cases whose time is measured.

A model whose 4-bit layers are served by the other products has layers that 4 bits hurt. Those stay in 8-bit integers, with a scale for
each token and each output channel, or in 16 bits. A converter rounds weights to int8 and takes them back. A server multiplies
activations by int8 weights, rounding the activations in the call, or multiplies what an earlier call rounded. A server of a mixture of
experts sorts the slots that its router chose by expert and multiplies every expert's tokens by that expert's own matrix, in int8 or
in 16 bits: groups of whatever sizes the router made.

Row lengths and row counts are those of the products measured beside this file (hidden size 5120, feed-forward width 17408) and generic
ones, odd ones among them; experts are a quarter of the hidden size wide.
"""
import math

import torch

own = False   # True: the framework's operators; False: the same mathematics in elementary torch operations

DEVICE = "cuda:0"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "int8": 1}


def _roundtrip(name, M, K, type_, out, acts="normal"):
    return {"name": name, "path": "roundtrip", "M": M, "K": K, "type": type_, "out": out, "acts": acts}


def _product(name, K, N, M, type_, acts="normal", given=False):
    """given: the activations are int8 with scales already, as an earlier call left them; type_ is the output's"""
    return {"name": name, "path": "product", "K": K, "N": N, "M": M, "type": type_, "acts": acts, "given": given}


def _sort(name, M, E, k, absent=0.0):
    return {"name": name, "path": "sort", "M": M, "E": E, "k": k, "absent": absent}


def _grouped(name, M, K, N, E, k, weights, type_, rows, absent=0.0, acts="normal"):
    """rows: "gather" reads the tokens' rows where they lie and writes in the order of the experts, "order" reads and writes in that
    order, "scatter" reads in that order and writes to the slots' places"""
    return {"name": name, "path": "grouped", "M": M, "K": K, "N": N, "E": E, "k": k, "weights": weights, "type": type_, "rows": rows,
            "absent": absent, "acts": acts}


def listed():
    return [
        # One token's activations to int8 and back: the smallest call of a tool that looks at what rounding does to them.
        _roundtrip("roundtrip_m1_k5120_bf16", 1, 5120, "bf16", "bf16", acts="outliers"),
        # A converter: a feed-forward tensor of fp32 weights, a scale per output channel.
        _roundtrip("roundtrip_m17408_k5120_fp32", 17408, 5120, "fp32", "fp32", acts="weights"),
        # One product of a decode step: the weights are the whole cost.
        _product("product_m1_k5120_n17408_bf16", 5120, 17408, 1, "bf16", acts="outliers"),
        # Some sequences decoded together, rows and lengths odd, activations that another product's call has rounded.
        _product("product_m13_k4099_n5121_fp16_given", 4099, 5121, 13, "fp16", acts="student_t", given=True),
        # A short prompt through the down projection, in fp32 as this framework's first products take and give it.
        _product("product_m201_k17408_n5120_fp32", 17408, 5120, 201, "fp32", acts="relu2"),
        # A prompt chunk through the feed-forward projection: the largest work.
        _product("product_m2048_k5120_n17408_bf16", 5120, 17408, 2048, "bf16"),
        # One decoded token's choices.
        _sort("sort_m1_e64_k8", 1, 64, 8),
        # A long prompt's choices among many experts, a few of them on another device.
        _sort("sort_m16384_e256_k8_absent", 16384, 256, 8, absent=0.125),
        # One decoded token through the up projection of its int8 experts.
        _grouped("grouped_m1_k5120_n1280_e64_k8_int8", 1, 5120, 1280, 64, 8, "int8", "bf16", "gather"),
        # An odd number of sequences decoded together through the down projection of 16-bit experts, some of them on another device.
        _grouped("grouped_m37_k1376_n4096_e60_k4_fp16_scatter", 37, 1376, 4096, 60, 4, "fp16", "fp16", "scatter", absent=0.25,
                 acts="relu2"),
        # A prompt chunk through the up projection of 16-bit experts: tokens read where they lie.
        _grouped("grouped_m2048_k5120_n1280_e64_k8_bf16", 2048, 5120, 1280, 64, 8, "bf16", "bf16", "gather"),
        # The same chunk through the down projection of int8 experts.
        _grouped("grouped_m2048_k1280_n5120_e64_k8_int8", 2048, 1280, 5120, 64, 8, "int8", "bf16", "order", acts="relu2"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.random()
    acts = rng.choice(("normal", "outliers", "student_t", "relu2"))
    if kind < 0.15:
        K = _log_int(rng, 32, 17408)
        M = _log_int(rng, 1, min(17408, 17408 * 5120 // K))
        c = _roundtrip("", M, K, rng.choice(tuple(TYPES)), rng.choice(("fp32", "bf16")), rng.choice((acts, "weights")))
    elif kind < 0.5:
        K = _log_int(rng, 256, 17408)
        N = _log_int(rng, 64, min(17408, 17408 * 5120 // K))
        c = _product("", K, N, _log_int(rng, 1, 2048), rng.choice(tuple(TYPES)), acts, rng.random() < 0.3)
    elif kind < 0.6:
        E = _log_int(rng, 4, 256)
        c = _sort("", _log_int(rng, 1, 16384), E, rng.randint(1, min(8, E)), rng.choice((0.0, 0.5)))
    else:
        E = rng.randint(4, 64)
        weights = rng.choice(("int8", "int8", "bf16", "fp16"))
        type_ = rng.choice(tuple(TYPES)) if weights == "int8" else weights
        K, N = _log_int(rng, 128, 5120), _log_int(rng, 128, 5120)
        N = min(N, 5120 * 1280 // K)
        c = _grouped("", _log_int(rng, 1, 2048), K, N, E, rng.randint(1, min(8, E)), weights, type_,
                     rng.choice(("gather", "order", "scatter")), rng.choice((0.0, 0.0, 0.5)), acts)
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
    """Codes [*shape, K] and scales [*shape] as a model file holds them: a gaussian row's largest element is about four deviations"""
    codes = torch.empty((*shape, K), dtype=torch.int8, device=DEVICE)
    flat = codes.view(-1, K)
    step = max(1, (1 << 26) // K)
    for i in range(0, flat.shape[0], step):
        rows = flat[i:i + step]
        rows.copy_((32.0 * torch.randn(rows.shape, device=DEVICE, generator=g)).round().clamp(-127, 127))
    scales = (0.5 + torch.rand(shape, device=DEVICE, generator=g)) * K ** -0.5 / 32
    return codes, scales


def _choices(case, g):
    """ids [M, k] of a router: experts differ in how often they are asked for, some are on another device"""
    M, E, k = case["M"], case["E"], case["k"]
    logits = 1.5 * torch.randn((M, E), device=DEVICE, generator=g) + 0.5 * torch.randn((E,), device=DEVICE, generator=g)
    ids = logits.topk(k, dim=1).indices.to(torch.int32)
    if case["absent"]:
        ids = torch.where(torch.rand((M, k), device=DEVICE, generator=g) < case["absent"], -1, ids)
    return ids


def _inputs(case, seed):
    g = _generator(seed)
    path, M = case["path"], case["M"]
    if path == "roundtrip":
        return {"x": _values(case["acts"], M, case["K"], g).to(TYPES[case["type"]])}
    if path == "sort":
        return {"ids": _choices(case, g)}
    K, N = case["K"], case["N"]
    if path == "product":
        codes, scales = _weight((N,), K, g)
        x = _values(case["acts"], M, K, g)
        s = {"codes": codes, "scales": scales}
        if case["given"]:
            s["x_scales"] = x.abs().amax(dim=1) / 127.0
            s["x"] = (x / s["x_scales"][:, None]).round().clamp(-127, 127).to(torch.int8)
        else:
            s["x"] = x.to(TYPES[case["type"]])
        return s
    E = case["E"]
    slots = M * case["k"]
    expert = _choices(case, g).flatten()
    expert = torch.where(expert < 0, E, expert)
    order = expert.sort(stable=True)
    ends = torch.searchsorted(order.values, torch.arange(E + 1, device=DEVICE, dtype=torch.int32))
    s = {"offsets": ends.to(torch.int32), "slots": order.indices.to(torch.int32), "expert": order.values}
    s["tokens"] = s["slots"] // case["k"]
    s["x"] = _values(case["acts"], M if case["rows"] == "gather" else slots, K, g).to(TYPES[case["type"]])
    if case["weights"] == "int8":
        s["codes"], s["scales"] = _weight((E, N), K, g)
    else:
        s["w"] = torch.empty((E, N, K), dtype=TYPES[case["weights"]], device=DEVICE)
        for e in range(E):
            s["w"][e] = torch.randn((N, K), device=DEVICE, generator=g) * K ** -0.5
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["path"] == "grouped":   # the buffer of a server's step; the rows of no group in it stay zeros
        state["out"] = torch.zeros((case["M"] * case["k"], case["N"]), dtype=TYPES[case["type"]], device=DEVICE)
    if own and case["path"] in ("product", "grouped"):   # what a server keeps: the weight's handle
        import ruquant_amd as rq
        state["weight"] = rq.I8Weight(state["codes"], state["scales"]) if "codes" in state else rq.HalfWeight(state["w"])
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _quantised(x):
    """codes (fp32) and scales of x [M, K]: the nearest whole numbers of x times the scale's reciprocal, ties to even. The product is
    taken in 64 bits, where it is exact: next to a tie its rounding to 32 would choose."""
    s = (x.float().abs().amax(dim=1) / 127.0).clamp_min(2.0 ** -126)
    r = 1.0 / s
    return (x.double() * r.double()[:, None]).round().float(), s


def _product_plain(s):
    case = s["case"]
    a, t = (s["x"].float(), s["x_scales"]) if case["given"] else _quantised(s["x"])
    y = a @ s["codes"].float().t()
    return (y * t[:, None] * s["scales"]).to(TYPES[case["type"]])


def _sort_plain(s):
    case = s["case"]
    E, k = case["E"], case["k"]
    expert = torch.where(s["ids"] < 0, E, s["ids"]).flatten()
    slots = expert.sort(stable=True).indices.to(torch.int32)
    counts = (expert[:, None] == torch.arange(E, device=DEVICE, dtype=torch.int32)).sum(dim=0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(dim=0)]).to(torch.int32)
    return offsets, slots, slots // k


def _grouped_plain(s):
    case = s["case"]
    E, N, K = case["E"], case["N"], case["K"]
    P = case["M"] * case["k"]
    if case["weights"] == "int8":
        x, t = _quantised(s["x"])
    else:
        x, t = s["x"].float(), None
    if case["rows"] == "gather":
        x = x[s["tokens"]]
        t = None if t is None else t[s["tokens"]]
    here = s["expert"] < E
    expert = torch.where(here, s["expert"], 0).long()
    w = s["codes"] if case["weights"] == "int8" else s["w"]
    if P <= E:   # few slots: the matrices of each slot's expert
        y = torch.bmm(w[expert].float(), x[:, :, None])[:, :, 0]
    else:        # many: each expert's rows side by side
        sizes = s["offsets"][1:] - s["offsets"][:-1]
        inside = torch.arange(P, device=DEVICE) - s["offsets"].long()[expert]
        inside = torch.where(here, inside, 0)
        side = torch.zeros((E, max(1, int(sizes.max())), K), device=DEVICE)
        at = here.nonzero()[:, 0]
        side[expert[at], inside[at]] = x[at]
        y = torch.bmm(side, w.float().transpose(1, 2).contiguous())[expert, inside]
    if t is not None:
        y = y * t[:, None] * s["scales"][expert]
    y = torch.where(here[:, None], y, 0.0).to(TYPES[case["type"]])
    if case["rows"] != "scatter":
        return y
    out = torch.zeros_like(y)
    out[s["slots"].long()] = y
    return out


def run(state):
    case = state["case"]
    path = case["path"]
    if not own:
        if path == "roundtrip":
            a, t = _quantised(state["x"])
            return (a * t[:, None]).to(TYPES[case["out"]])
        return {"product": _product_plain, "sort": _sort_plain, "grouped": _grouped_plain}[path](state)
    import ruquant_amd as rq
    if path == "roundtrip":
        codes, scales = rq.i8_quantize(state["x"])
        return rq.i8_dequantize(codes, scales, dtype=TYPES[case["out"]])
    if path == "product":
        if case["given"]:
            return rq.i8_mul_mat(state["weight"], state["x"], scales=state["x_scales"], dtype=TYPES[case["type"]])
        return rq.i8_mul_mat(state["weight"], state["x"])
    if path == "sort":
        return rq.sort_slots(state["ids"], case["E"])
    rows = state["tokens"] if case["rows"] == "gather" else None
    out_rows = state["slots"] if case["rows"] == "scatter" else None
    return rq.grouped_mul_mat(state["weight"], state["x"], state["offsets"], rows=rows, out_rows=out_rows, out=state["out"])


def work(case):
    path, M = case["path"], case["M"]
    if path == "sort":
        slots = M * case["k"]
        return {"bytes": 12 * slots + 4 * (case["E"] + 1), "flops": slots}
    K = case["K"]
    size = BYTES[case["type"]]
    if path == "roundtrip":   # (the codes in between are written and read once, by two calls)
        return {"bytes": M * K * (size + BYTES[case["out"]] + 2) + 8 * M, "flops": 4 * M * K}
    N = case["N"]
    if path == "product":
        return {"bytes": N * (K + 4) + M * (K * (1 if case["given"] else size) + N * size) + (4 * M if case["given"] else 0),
                "flops": 2 * M * N * K}
    E, k = case["E"], case["k"]
    share = 1.0 - case["absent"]
    slots = share * M * k
    asked = E * (1.0 - (1.0 - share * k / E) ** M)   # experts that some token asks for, were all asked for equally often
    read = min(M, slots) if case["rows"] == "gather" else slots
    weight = N * (K + 4) if case["weights"] == "int8" else 2 * N * K
    return {"bytes": int(asked * weight + size * (read * K + slots * N) + 4 * slots * (case["rows"] != "order")) + 4 * (E + 1),
            "flops": int(2 * slots * N * K)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _rounded64(x):
    """(codes, scales) in 64 bits. A scale is an fp32 number, as the operator gives it, and so is the reciprocal that the elements are
    multiplied by; nothing else is rounded but to the codes."""
    v = x.double()
    s = torch.clamp(v.abs().max(dim=1, keepdim=True).values / 127, min=2.0 ** -126).float().double()
    return torch.round(v * torch.reciprocal(s).float().double()), s


def exact(case, seed):
    path = case["path"]
    if path == "sort":
        return None   # (whole numbers)
    s = _inputs(case, seed)
    if path == "roundtrip":
        a, t = _rounded64(s["x"])
        return a * t
    if path == "product":
        a, t = (s["x"].double(), s["x_scales"].double()[:, None]) if case["given"] else _rounded64(s["x"])
        return torch.matmul(a, s["codes"].double().T.contiguous()) * t * s["scales"].double()[None, :]
    y = torch.zeros((case["M"] * case["k"], case["N"]), dtype=torch.float64, device=DEVICE)
    offsets = s["offsets"].tolist()
    for e in range(case["E"]):
        p = torch.arange(offsets[e], offsets[e + 1], device=DEVICE)
        if not len(p):
            continue
        x = s["x"][s["tokens"][p].long() if case["rows"] == "gather" else p]
        if case["weights"] == "int8":
            a, t = _rounded64(x)
            part = torch.matmul(a, s["codes"][e].double().T.contiguous()) * t * s["scales"][e].double()[None, :]
        else:
            part = torch.matmul(x.double(), s["w"][e].double().T.contiguous())
        y[s["slots"][p].long() if case["rows"] == "scatter" else p] = part
    return y
