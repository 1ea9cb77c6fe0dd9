"""The operators of a feed-forward in 8-bit floating point (e4m3 values, a 32-bit scale for each block of 128), for timing them and for
comparing their results: the norm in front that leaves quantised rows (`norm`), the gated activation that does (`glu`), the product of such
rows with such weights (`linear`), the router that chooses experts by groups (`route`) and the experts' products (`experts`).

What is quantised: row t of an activation has a scale for each 128 columns, s = max(max |v| / 448, 2^-126), and holds e4m3(v / s); a matrix
[rows][cols] has a scale for each 128 x 128 block.  Columns come in sixteens; the last block of a row or a matrix may be a part of one.

With `own` False `run` computes an operator from elementary torch operations, with `own` True through the framework's calls.
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
BLOCK = 128
TINY = 2.0 ** -126
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IDS = {"f32": 0, "f16": 1, "bf16": 2}          # the framework's ids of these types


def listed():
    return [
        # the norm in front of a decode step's feed-forward: one token, where latency counts
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 2048, "type": "f32", "add": True, "plain": True},
        # a long prompt's residual update, norm and quantisation, 32-bit residual stream
        {"name": "norm_prompt", "kind": "norm", "rows": 4096, "cols": 4096, "type": "f32", "add": True, "plain": False},
        # the activation of a few users' tokens, halves, a width that ends inside a block
        {"name": "glu_batch", "kind": "glu", "rows": 9, "cols": 2832, "type": "f16", "act": 0},
        # the activation of a long prompt of odd length
        {"name": "glu_prompt", "kind": "glu", "rows": 2051, "cols": 11008, "type": "bf16", "act": 0},
        # a decode step's output product: one token, added into the residual
        {"name": "linear_token", "kind": "linear", "tokens": 1, "rows": 4096, "cols": 11008, "type": "f32", "accumulate": True, "bias": False},
        # a batch of users, biases, a matrix that ends inside a block both ways
        {"name": "linear_batch", "kind": "linear", "tokens": 24, "rows": 5632, "cols": 2064, "type": "f16", "accumulate": False, "bias": True},
        # a long prompt: the matrix cores' rate
        {"name": "linear_prompt", "kind": "linear", "tokens": 4096, "rows": 11008, "cols": 4096, "type": "bf16", "accumulate": False, "bias": False},
        # a batch of users' tokens to 64 experts in 8 groups
        {"name": "route_batch", "kind": "route", "rows": 13, "experts": 64, "groups": 8, "kept": 3, "best": 2, "top": 6, "scores": 1, "renorm": True, "masked": 0},
        # a long prompt's tokens to 256 experts
        {"name": "route_prompt", "kind": "route", "rows": 8191, "experts": 256, "groups": 8, "kept": 4, "best": 2, "top": 8, "scores": 1, "renorm": True, "masked": 0},
        # one token's experts
        {"name": "experts_token", "kind": "experts", "rows": 1, "width": 2048, "ff": 1408, "experts": 64, "top": 6, "type": "bf16", "accumulate": False, "act": 0, "dropped": 0.0},
        # a batch of users' tokens: a few rows for every expert
        {"name": "experts_batch", "kind": "experts", "rows": 53, "width": 2048, "ff": 704, "experts": 32, "top": 4, "type": "bf16", "accumulate": False, "act": 0, "dropped": 0.0},
        # a long prompt of odd length, some choices dropped for want of room
        {"name": "experts_prompt", "kind": "experts", "rows": 3001, "width": 2048, "ff": 1408, "experts": 64, "top": 6, "type": "bf16", "accumulate": False, "act": 0, "dropped": 0.05},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    most = max(cost(c) for c in listed())
    while True:
        kind = rng.choice(["norm", "glu", "linear", "route", "experts"])
        kinds = rng.choice(list(TYPES))
        if kind == "norm":
            c = {"rows": log(1, 8192), "cols": 16 * log(4, 1024), "type": kinds, "add": rng.random() < 0.7, "plain": rng.random() < 0.5}
        elif kind == "glu":
            c = {"rows": log(1, 8192), "cols": 16 * log(4, 1024), "type": kinds, "act": rng.choice([0, 1, 2, 3, 4])}
        elif kind == "linear":
            c = {"tokens": log(1, 4096), "rows": log(48, 16384), "cols": 16 * log(4, 1024), "type": kinds, "accumulate": rng.random() < 0.3, "bias": rng.random() < 0.3}
        elif kind == "route":
            groups, each = rng.choice([1, 2, 4, 8, 12]), rng.choice([2, 4, 8, 15, 16, 32])
            kept = rng.randint(1, groups)
            c = {"rows": log(1, 16384), "experts": groups * each, "groups": groups, "kept": kept, "best": rng.choice([1, 2]), "top": rng.randint(1, min(16, kept * each)),
                 "scores": rng.choice([0, 1]), "renorm": rng.random() < 0.7, "masked": rng.choice([0, 0, 1])}
        else:
            experts = rng.choice([4, 8, 16, 32, 60, 64])
            c = {"rows": log(1, 3000), "width": 16 * log(16, 256), "ff": 16 * log(8, 128), "experts": experts, "top": rng.randint(1, min(8, experts)), "type": rng.choice(["f16", "bf16"]),
                 "accumulate": rng.random() < 0.3, "act": rng.choice([0, 1, 3]), "dropped": rng.choice([0.0, 0.0, 0.1])}
        c["kind"] = kind
        if cost(c) <= most:
            return c


def cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def size(c):
    return TYPES[c["type"]].itemsize


def work(case):
    c, blocks = case, lambda n: -(-n // BLOCK)
    if c["kind"] == "norm":
        values = c["rows"] * c["cols"]
        return {"bytes": values * (size(c) * (1 + (2 if c["add"] else 0) + (1 if c["plain"] else 0)) + 1) + c["rows"] * blocks(c["cols"]) * 4 + 2 * c["cols"], "flops": 6 * values}
    if c["kind"] == "glu":
        values = c["rows"] * c["cols"]
        return {"bytes": values * (size(c) * (2 if c["act"] < 4 else 1) + 1) + c["rows"] * blocks(c["cols"]) * 4, "flops": 10 * values}
    if c["kind"] == "linear":
        t, n, k = c["tokens"], c["rows"], c["cols"]
        return {"bytes": n * k + t * k + 4 * blocks(k) * (blocks(n) + t) + t * n * size(c) * (2 if c["accumulate"] else 1), "flops": 2 * t * n * k}
    if c["kind"] == "route":
        return {"bytes": c["rows"] * (4 * c["experts"] + 8 * c["top"]) + 4 * c["experts"], "flops": 20 * c["rows"] * c["experts"]}
    pairs = c["rows"] * c["top"] * (1 - c["dropped"])
    met = c["experts"] * (1 - (1 - 1 / c["experts"]) ** pairs)          # experts that a step meets, choices taken as independent
    return {"bytes": met * 3 * c["width"] * c["ff"] + c["rows"] * (c["width"] * (1 + size(c) * (2 if c["accumulate"] else 1)) + 4 * blocks(c["width"]) + 8 * c["top"]),
            "flops": 6 * pairs * c["width"] * c["ff"]}


# ---------------------------------------------------------------- inputs
def spread(scale, rows, cols):
    """a matrix's block scales for each of its values"""
    return scale.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def rows_scale(scale, cols):
    """a row's scales for each of its columns"""
    return scale.repeat_interleave(BLOCK, -1)[..., :cols]


def padded(v, n, dim):
    shape = list(v.shape)
    shape[dim] = n - shape[dim]
    return torch.cat([v, v.new_zeros(shape)], dim) if shape[dim] else v


def quantised_rows(v):
    """(e4m3 rows, scales) of 32-bit rows"""
    cols = v.shape[-1]
    blocks = -(-cols // BLOCK)
    most = padded(v, blocks * BLOCK, v.dim() - 1).unflatten(-1, (blocks, BLOCK)).abs().amax(-1)
    scale = (most / 448).clamp_min(TINY)
    return (v / rows_scale(scale, cols)).to(F8), scale


def matrices(count, rows, cols, std, g):
    """`count` matrices [rows][cols] in e4m3 with their block scales, as a checkpoint holds them"""
    br, bc = -(-rows // BLOCK), -(-cols // BLOCK)
    w = torch.randn(count, rows, cols, generator=g, device="cuda") * (std * (0.5 + torch.rand(count, rows, 1, generator=g, device="cuda")))
    scales = padded(padded(w, br * BLOCK, 1), bc * BLOCK, 2).view(count, br, BLOCK, bc, BLOCK).abs().amax((2, 4)) / 448
    return w.div_(spread(scales, rows, cols)).to(F8), scales


def made(*shape, kind=F8):
    return torch.empty(*shape, dtype=kind, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    s = {"case": c, "stream": torch.cuda.current_stream().cuda_stream}
    blocks = lambda n: -(-n // BLOCK)  # noqa: E731
    if c["kind"] == "norm":
        rows, cols, kind = c["rows"], c["cols"], TYPES[c["type"]]
        # a residual stream: rows of unlike size, a few columns that stand out; a sub-layer's output to add
        s["x"] = (normal(rows, cols) * (0.5 + 3 * torch.rand(rows, 1, generator=g, device="cuda")) * (1 + 20 * (torch.rand(cols, generator=g, device="cuda") < 0.005))).to(kind)
        s["m"] = (0.3 * normal(rows, cols)).to(kind) if c["add"] else None
        s["w"] = (1 + 0.1 * normal(cols)).to(torch.bfloat16)
        s["h"] = made(rows, cols, kind=kind) if c["plain"] else None
        s["q"], s["scale"] = made(rows, cols), made(rows, blocks(cols), kind=torch.float32)
        return s
    if c["kind"] == "glu":
        rows, cols, kind = c["rows"], c["cols"], TYPES[c["type"]]
        s["gu"] = (2 * normal(rows, cols * (2 if c["act"] < 4 else 1))).to(kind)
        s["q"], s["scale"] = made(rows, cols), made(rows, blocks(cols), kind=torch.float32)
        return s
    if c["kind"] == "linear":
        s["a"], s["sa"] = quantised_rows(normal(c["tokens"], c["cols"]))
        q, sw = matrices(1, c["rows"], c["cols"], 0.02, g)
        s["w"], s["sw"] = q[0], sw[0]
        s["bias"] = (0.1 * normal(c["rows"])).to(torch.bfloat16) if c["bias"] else None
        s["c"] = normal(c["tokens"], c["rows"]).to(TYPES[c["type"]])
        s["ws"] = made(64 << 20, kind=torch.uint8)
        return s
    if c["kind"] == "route":
        s["logits"] = 1.5 * normal(c["rows"], c["experts"])
        s["corr"] = 0.05 * normal(c["experts"])
        if c["masked"]:          # experts that a row may not use, and rows that may use none
            s["logits"][torch.rand(c["rows"], c["experts"], generator=g, device="cuda") < 0.3] = -math.inf
            s["logits"][torch.rand(c["rows"], generator=g, device="cuda") < 0.05] = -math.inf
        s["idx"], s["wgt"] = made(c["rows"], c["top"], kind=torch.int32), made(c["rows"], c["top"], kind=torch.float32)
        return s
    rows, width, ff, experts, top = c["rows"], c["width"], c["ff"], c["experts"], c["top"]
    s["a"], s["sa"] = quantised_rows(normal(rows, width))
    # gate and up of an expert lie behind each other, each with blocks of its own
    q, sc = matrices(2 * experts, ff, width, 1.5 * width ** -0.5, g)
    s["gu"], s["sgu"] = q.view(experts, 2, ff, width), sc.view(experts, 2, blocks(ff), blocks(width))
    s["down"], s["sdown"] = matrices(experts, width, ff, ff ** -0.5, g)
    liked = 0.3 * normal(experts)          # some experts are met more often than others
    s["idx"] = (normal(rows, experts) + liked).argsort(-1, descending=True)[:, :top].to(torch.int32).contiguous()
    s["wgt"] = torch.rand(rows, top, generator=g, device="cuda") + 0.1
    s["wgt"] /= s["wgt"].sum(-1, keepdim=True)
    s["idx"][torch.rand(rows, top, generator=g, device="cuda") < c["dropped"]] = -1
    s["most"] = max(1, int(torch.bincount(s["idx"][s["idx"] >= 0].flatten().long(), minlength=experts).max()))          # rows that the most liked expert gets
    s["y"] = normal(rows, width).to(TYPES[c["type"]])
    s["ws"] = made(workspace_bytes(c), kind=torch.uint8)
    return s


def workspace_bytes(c):
    """room for the experts' rows between the products, and some for their lists"""
    pairs = c["rows"] * c["top"]
    return (pairs + 64 * c["experts"] + 256) * (4 * (c["width"] + 2 * c["ff"]) + 64) + (16 << 20)


# ---------------------------------------------------------------- the plain forms, in 32 bits
def gated(act, gate, up):
    if act == 3:
        g, u = gate.clamp_max(7.0), up.clamp(-7.0, 7.0)
        return g / (1 + torch.exp(-1.702 * g)) * (u + 1)
    if act == 0:
        return gate / (1 + torch.exp(-gate)) * up
    if act == 1:
        return 0.5 * gate * (1 + torch.tanh(0.7978845608028654 * (gate + 0.044715 * gate ** 3))) * up
    return gate.clamp_min(0) * up


def plain_norm(s):
    if s["m"] is not None:
        s["x"].copy_(s["x"].float() + s["m"].float())
    x = s["x"].float()
    h = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["w"].float()
    q, scale = quantised_rows(h)
    return {"x": s["x"], "q": q, "scale": scale, "h": None if s["h"] is None else h.to(s["x"].dtype)}


def plain_glu(s):
    c, v = s["case"], s["gu"].float()
    q, scale = quantised_rows(v if c["act"] == 4 else gated(c["act"], v[:, :c["cols"]], v[:, c["cols"]:]))
    return {"q": q, "scale": scale}


def plain_linear(s):
    c = s["case"]
    a = s["a"].float() * rows_scale(s["sa"], c["cols"])
    w = s["w"].float() * spread(s["sw"], c["rows"], c["cols"])
    y = a @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return s["c"].copy_(s["c"].float() + y if c["accumulate"] else y)


def plain_route(s):
    c = s["case"]          # in 64 bits: a choice at the border must not hang on a rounding
    z = s["logits"].double()
    may = z > -math.inf
    if c["scores"] == 1:
        score = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e300))
        score = e / e.sum(-1, keepdim=True)
    choice = torch.where(may, score + s["corr"].double(), -math.inf)
    each = c["experts"] // c["groups"]
    best = choice.view(-1, c["groups"], each).sort(-1, descending=True).values[..., :c["best"]]
    of_group = torch.where(best[..., 0] > -math.inf, torch.where(best > -math.inf, best, 0.0).sum(-1), -math.inf)
    kept = of_group.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
    keep = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, kept, True)
    choice = torch.where(keep.repeat_interleave(each, 1), choice, -math.inf)
    value, idx = choice.sort(dim=-1, descending=True, stable=True)
    value, idx = value[:, :c["top"]], idx[:, :c["top"]]
    wgt = torch.where(value > -math.inf, score.gather(1, idx), 0.0)
    if c["renorm"]:
        den = wgt.sum(-1, keepdim=True) + 1e-20
        wgt = torch.where(den > 0, wgt / den, 0.0) * 2.5
    return {"idx": torch.where(value > -math.inf, idx, -1).int(), "wgt": wgt.float()}


def plain_experts(s):
    c = s["case"]
    width, ff, experts, top = c["width"], c["ff"], c["experts"], c["top"]
    a = s["a"].float() * rows_scale(s["sa"], width)
    pairs = s["idx"].flatten().long()
    wgt = torch.where(pairs >= 0, s["wgt"].flatten(), 0.0)
    row = torch.arange(len(pairs), device="cuda") // top
    if len(pairs) <= experts:          # few pairs: each its own expert's matrices
        e = pairs.clamp_min(0)
        rows = a[row].unsqueeze(1)
        gu, sgu, down, sdown = s["gu"].view(torch.uint8)[e].view(F8), s["sgu"][e], s["down"].view(torch.uint8)[e].view(F8), s["sdown"][e]
    else:          # many: the pairs of an expert together, with room for those of the most liked one
        e = torch.where(pairs >= 0, pairs, experts)
        order = e.sort(stable=True).indices
        count = torch.zeros(experts + 1, dtype=torch.long, device="cuda").scatter_add_(0, e, torch.ones_like(e))
        place = torch.empty_like(e)
        place[order] = torch.arange(len(e), device="cuda") - (count.cumsum(0) - count)[e[order]]
        at = torch.where(pairs >= 0, pairs * s["most"] + place, experts * s["most"])
        rows = a.new_zeros(experts * s["most"] + 1, width)
        rows[at] = a[row]
        rows = rows[:-1].view(experts, s["most"], width)
        gu, sgu, down, sdown = s["gu"], s["sgu"], s["down"], s["sdown"]
    gate, up = (torch.bmm(rows, (gu[:, i].float() * spread(sgu[:, i], ff, width)).transpose(1, 2)) for i in (0, 1))
    q, scale = quantised_rows(gated(c["act"], gate, up))
    y = torch.bmm(q.float() * rows_scale(scale, ff), (down.float() * spread(sdown, width, ff)).transpose(1, 2)).view(-1, width)
    if len(pairs) > experts:
        y = y[at.clamp_max(len(y) - 1)]
    y = (y * wgt.unsqueeze(1)).view(-1, top, width).sum(1)
    return s["y"].copy_(s["y"].float() + y if c["accumulate"] else y)


# ---------------------------------------------------------------- the framework's calls
_library = None


def library():
    global _library
    if _library is None:
        from inferflow_amd import check, lib
        _library = lib(), check
    return _library


def at(t):
    return None if t is None else t.data_ptr()


def own_norm(s):
    c = s["case"]
    L, check = library()
    n = c["cols"]
    check(L.ifa_norm_add_fp8(IDS[c["type"]], at(s["x"]), n, c["rows"], n, at(s["m"]), n, at(s["w"]), 0.0, 1e-6, at(s["h"]), n, at(s["q"]), n, at(s["scale"]), s["scale"].shape[1], s["stream"]))
    return {"x": s["x"], "q": s["q"], "scale": s["scale"], "h": s["h"]}


def own_glu(s):
    c = s["case"]
    L, check = library()
    check(L.ifa_glu_fp8(c["act"], 7.0, IDS[c["type"]], at(s["gu"]), s["gu"].shape[1], c["rows"], c["cols"], at(s["q"]), c["cols"], at(s["scale"]), s["scale"].shape[1], s["stream"]))
    return {"q": s["q"], "scale": s["scale"]}


def own_linear(s):
    c = s["case"]
    L, check = library()
    check(L.ifa_linear_fp8(at(s["w"]), at(s["sw"]), c["rows"], c["cols"], at(s["a"]), c["cols"], at(s["sa"]), s["sa"].shape[1], c["tokens"], at(s["bias"]), int(c["accumulate"]),
                           IDS[c["type"]], at(s["c"]), c["rows"], at(s["ws"]), s["ws"].numel(), s["stream"]))
    return s["c"]


def own_route(s):
    c = s["case"]
    L, check = library()
    check(L.ifa_moe_route_groups_f32(c["scores"], c["groups"], c["kept"], c["best"], int(c["renorm"]), 1e-20, 2.5 if c["renorm"] else 1.0, at(s["logits"]), c["experts"], c["rows"],
                                     c["experts"], c["top"], at(s["corr"]), at(s["idx"]), at(s["wgt"]), s["stream"]))
    return {"idx": s["idx"], "wgt": s["wgt"]}


def own_experts(s):
    c = s["case"]
    L, check = library()
    check(L.ifa_moe_experts_fp8(c["act"], 7.0, at(s["a"]), c["width"], at(s["sa"]), s["sa"].shape[1], c["rows"], c["width"], c["ff"], c["experts"], c["top"], at(s["gu"]), at(s["sgu"]),
                                at(s["down"]), at(s["sdown"]), at(s["idx"]), at(s["wgt"]), at(s["ws"]), s["ws"].numel(), IDS[c["type"]], at(s["y"]), c["width"], int(c["accumulate"]),
                                s["stream"]))
    return s["y"]


def run(state):
    if own:
        return {"norm": own_norm, "glu": own_glu, "linear": own_linear, "route": own_route, "experts": own_experts}[state["case"]["kind"]](state)
    return {"norm": plain_norm, "glu": plain_glu, "linear": plain_linear, "route": plain_route, "experts": plain_experts}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- the definition in 64 bits
def e4m3(v):
    """the nearest value with four significant bits, an exponent of -6 at least and a size of 448 at most (ties to the even one)"""
    _, e = torch.frexp(v)
    step = ((e.clamp_min(-5) - 4 + 1023).long() << 52).view(torch.float64)          # (2^(e - 4), exactly)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def in_blocks(v):
    """(e4m3 values, scales) of 64-bit rows, block by block"""
    parts = [(p, (p.abs().amax(-1, keepdim=True) / 448).clamp_min(TINY)) for p in v.split(BLOCK, -1)]
    return torch.cat([e4m3(p / t) for p, t in parts], -1), torch.cat([t for _, t in parts], -1)


def blocks_product(a, sa, w, sw):
    """rows a (values, scales) times the transpose of matrix w (values, scales)"""
    n = w.shape[0]
    of_row = torch.arange(n, device=w.device) // BLOCK
    return sum(a[:, k:k + BLOCK].double() @ w[:, k:k + BLOCK].double().t() * sa[:, k // BLOCK, None].double() * sw[of_row, k // BLOCK].double() for k in range(0, w.shape[1], BLOCK))


def sigma(z):
    return torch.special.expit(z)


def gate_exact(act, g, u):
    if act == 0:
        return g * sigma(g) * u
    if act == 1:
        return g * sigma(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u          # (1 + tanh z) / 2 = sigma(2 z)
    if act == 2:
        return torch.relu(g) * u
    g, u = torch.clamp(g, max=7.0), torch.clamp(u, -7.0, 7.0)
    return g * sigma(1.702 * g) * (u + 1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "norm":
        x = s["x"].double()
        if c["add"]:
            x = (x + s["m"].double()).to(s["x"].dtype).double()          # (the stored row is what is normed)
        h = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / c["cols"] + 1e-6) * s["w"].double()
        q, scale = in_blocks(h)
        return {"x": x, "q": q, "scale": scale, "h": h if c["plain"] else None}
    if c["kind"] == "glu":
        v = s["gu"].double()
        q, scale = in_blocks(v if c["act"] == 4 else gate_exact(c["act"], *v.chunk(2, -1)))
        return {"q": q, "scale": scale}
    if c["kind"] == "linear":
        y = blocks_product(s["a"], s["sa"], s["w"], s["sw"])
        y = y + (s["bias"].double() if c["bias"] else 0.0)
        return y + s["c"].double() if c["accumulate"] else y
    if c["kind"] == "route":          # by repeated first maxima
        z, corr = s["logits"].double(), s["corr"].double()
        score = sigma(z) if c["scores"] == 1 else torch.nan_to_num(torch.softmax(z, -1))
        left = torch.where(z == -math.inf, -math.inf, score + corr)
        each = c["experts"] // c["groups"]
        g = left.unflatten(1, (c["groups"], each)).clone()
        total = torch.zeros(c["rows"], c["groups"], dtype=torch.float64, device="cuda")
        none = g.amax(-1) == -math.inf
        for _ in range(c["best"]):
            v, i = g.max(-1)
            total += torch.where(v == -math.inf, 0.0, v)
            g.scatter_(2, i[..., None], -math.inf)
        total[none] = -math.inf
        open_ = torch.zeros_like(none)
        order = torch.arange(c["groups"], device="cuda")
        for i in range(c["groups"]):          # a group is kept if fewer than `kept` are better (the lower index wins a tie)
            better = (total > total[:, i:i + 1]) | ((total == total[:, i:i + 1]) & (order < i))
            open_[:, i] = better.sum(-1) < c["kept"]
        left = torch.where(open_.repeat_interleave(each, 1), left, -math.inf)
        idx, wgt = [], []
        place = torch.arange(c["experts"], device="cuda")
        for _ in range(c["top"]):
            v = left.amax(-1)
            first = torch.where(left == v[:, None], place, c["experts"]).amin(-1)
            none = v == -math.inf
            idx.append(torch.where(none, -1, first))
            wgt.append(torch.where(none, 0.0, score.gather(1, first[:, None])[:, 0]))
            left.scatter_(1, first[:, None], -math.inf)
        wgt = torch.stack(wgt, 1)
        if c["renorm"]:
            wgt = 2.5 * wgt / (wgt.sum(1, keepdim=True) + 1e-20)
        return {"idx": torch.stack(idx, 1).int(), "wgt": wgt}
    y = torch.zeros(c["rows"], c["width"], dtype=torch.float64, device="cuda")
    for e in range(c["experts"]):
        t, k = (s["idx"] == e).nonzero(as_tuple=True)
        if len(t):
            gate, up = (blocks_product(s["a"].float()[t], s["sa"][t], s["gu"][e, i], s["sgu"][e, i]) for i in (0, 1))
            v = blocks_product(*in_blocks(gate_exact(c["act"], gate, up)), s["down"][e], s["sdown"][e])
            y.index_add_(0, t, v * s["wgt"][t, k].double()[:, None])
    return y + s["y"].double() if c["accumulate"] else y
