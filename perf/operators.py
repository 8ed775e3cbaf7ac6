"""Routing by scores and the 8-bit products with a scale per token and per channel, as a MoE block with int8
weights runs them: the calls that performance work on these operators is measured on.

A case names one operator and its sizes:

  route   logits [M][E] -> the k experts of each token and their weights (`route_scores`)
  quant   x [M][K] -> int8 rows with a scale each (`quantize_rows`)
  gemm    int8 rows x an int8 matrix [R][K] -> [M][R] (`gemm_i8`)
  up      each token through its k experts' gate and up products and SwiGLU -> [M * k][F] (`experts_plan`,
          `experts_up_i8`)
  down    the activation rows through their experts' down products, weighted and summed per token -> [M][H]
          (`experts_plan`, `experts_down_i8`)

M tokens, E experts of width F, hidden size H.  dtype: of x in `quant`, of the output elsewhere.  spare: values behind
each row of x that belong to something else (a slice of a wider tensor).  skew: an expert's load falls as
1 / (rank + 1)^skew.  ragged: a token takes 1 to k experts, as routing by mass gives them.  mask: the share of the
experts that a token may not take.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
SLOTS = 32  # experts a row of ids and weights has room for
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TILE = 64   # entries of one expert that the plain form multiplies together


def _package():
    """This repository's package, as a program has it imported once."""
    if "trmoe" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tr-infer_amd"))
        import trmoe  # noqa: F401
    return sys.modules["trmoe"]


# ---- the cases -------------------------------------------------------------------------------------

def _route(M, E, k, score, bias=True, groups=1, keep=1, group_top=2, renorm=True, factor=1.0, mask=0.0, **more):
    return dict(more, op="route", M=M, E=E, k=k, score=score, bias=bias, groups=groups, keep=keep,
                group_top=group_top, renorm=renorm, factor=factor, mask=mask)


def _quant(M, K, dtype, spare=0, **more):
    return dict(more, op="quant", M=M, K=K, dtype=dtype, spare=spare)


def _gemm(M, R, K, dtype, bias=False, **more):
    return dict(more, op="gemm", M=M, R=R, K=K, dtype=dtype, bias=bias)


def _experts(op, M, k, E, H, F, dtype, skew=0.0, ragged=False, **more):
    return dict(more, op=op, M=M, k=k, E=E, H=H, F=F, dtype=dtype, skew=skew, ragged=ragged)


def listed():
    return [
        # one decoded token: sigmoid scores, a balance bias, 4 of 8 groups
        _route(1, 256, 8, "sigmoid", groups=8, keep=4, factor=2.5, name="route_decode"),
        # a prompt on the layer's own shape: softmax over 512 experts, some of them not to be taken
        _route(2048, 512, 10, "softmax", bias=False, mask=0.1, name="route_prompt"),
        # a large prefill
        _route(16384, 256, 8, "sigmoid", groups=8, keep=4, factor=2.5, name="route_prefill"),
        # the rows of a few decoded tokens
        _quant(4, 2048, "f32", name="quant_decode"),
        # the rows of a large prefill, a slice of a wider projection's output
        _quant(8192, 4096, "bf16", spare=1024, name="quant_prefill"),
        # a dense projection of one decoded token: the weights are read once
        _gemm(1, 12288, 2560, "f32", name="gemm_decode"),
        # a short prompt, nothing a multiple of anything
        _gemm(77, 5003, 1999, "f16", bias=True, name="gemm_ragged"),
        # the same projection in a large prefill
        _gemm(4096, 12288, 2560, "bf16", name="gemm_prefill"),
        # one decoded token through its ten experts
        _experts("up", 1, 10, 512, 2048, 512, "f32", name="up_decode"),
        # a prompt on fewer, wider experts, unevenly loaded
        _experts("up", 2000, 8, 128, 2048, 768, "bf16", skew=0.5, name="up_prefill"),
        # four sequences' tokens through the down products
        _experts("down", 4, 10, 512, 2048, 512, "f32", name="down_decode"),
        # a large prefill
        _experts("down", 4096, 10, 512, 2048, 512, "f32", skew=0.3, name="down_prefill"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "quant", "gemm", "gemm", "up", "up", "down", "down"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = _log(rng, 4, 512 // groups)
        keep = rng.randint(1, groups)
        return _route(_log(rng, 1, 16384), groups * size, rng.randint(1, min(16, keep * size)),
                      rng.choice(["sigmoid", "softmax"]), bias=rng.random() < 0.6, groups=groups, keep=keep,
                      group_top=rng.choice([1, 2]), renorm=rng.random() < 0.7, factor=rng.choice([1.0, 2.5]),
                      mask=rng.choice([0.0, 0.0, 0.3]))
    if op == "quant":
        K = _log(rng, 32, 12288)
        return _quant(_log(rng, 1, min(8192, 8192 * 4096 // K)), K, rng.choice(list(DTYPES)),
                      spare=rng.choice([0, 0, 8, 96, 1]))
    if op == "gemm":
        R, K = _log(rng, 64, 16384), _log(rng, 64, 12288)
        return _gemm(_log(rng, 1, min(4096, 4096 * 12288 * 2560 // (R * K))), R, K, rng.choice(list(DTYPES)),
                     bias=rng.random() < 0.5)
    E, H, F = _log(rng, 8, 512), _log(rng, 256, 2560), _log(rng, 64, 1024)
    while E * H * F > 512 * 2048 * 512:
        E //= 2
    k = rng.randint(1, min(10, E))
    M = _log(rng, 1, 4096)
    while M * k * H * F > 4096 * 10 * 2048 * 512:
        M = (M + 1) // 2
    return _experts(op, M, k, E, H, F, rng.choice(list(DTYPES)), skew=rng.choice([0.0, 0.3, 0.8]),
                    ragged=rng.random() < 0.3)


# ---- inputs ----------------------------------------------------------------------------------------

def _pad16(n):
    return (n + 15) // 16 * 16


def _i8(gen, *shape):
    """int8 values as quantised rows hold them (a normal cut at 127, near four deviations), the rows a multiple of 16
    bytes apart."""
    *lead, k = shape
    q = torch.empty((*lead, _pad16(k)), dtype=torch.int8, device=DEV)
    flat = q.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.randn(part.numel(), device=DEV, generator=gen).mul_(32.0).round_().clamp_(-127, 127))
    return q[..., :k]


def _scales(gen, *shape, around):
    return torch.empty(shape, device=DEV).uniform_(0.5 * around, 1.5 * around, generator=gen)


def _routing(gen, c):
    """ids and weights as a router leaves them: k distinct experts a token, best first, in rows of SLOTS."""
    M, E, k = c["M"], c["E"], c["k"]
    load = torch.arange(1, E + 1, device=DEV, dtype=torch.float32).pow(-c["skew"]).log()
    load = load[torch.randperm(E, device=DEV, generator=gen)]
    noise = -torch.rand((M, E), device=DEV, generator=gen).clamp_min(1e-20).log_().neg_().log_()  # Gumbel: draws without replacement
    ids = torch.full((M, SLOTS), -1, dtype=torch.int32, device=DEV)
    ids[:, :k] = (noise + load).topk(k, dim=1).indices
    w = torch.zeros((M, SLOTS), device=DEV)
    w[:, :k] = torch.randn((M, k), device=DEV, generator=gen).softmax(1).sort(dim=1, descending=True).values
    n = torch.randint(1, k + 1, (M,), device=DEV, generator=gen) if c["ragged"] else torch.full((M,), k, device=DEV)
    return ids, w, n.to(torch.int32)


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    M = c["M"]
    if c["op"] == "route":
        logits = torch.randn((M, c["E"]), device=DEV, generator=gen) * 1.3
        if c["mask"]:
            out = torch.rand((M, c["E"]), device=DEV, generator=gen) < c["mask"]
            logits.masked_fill_(out, -math.inf)
        bias = torch.randn(c["E"], device=DEV, generator=gen) * 0.05 if c["bias"] else None
        return {"logits": logits, "bias": bias}
    if c["op"] == "quant":
        wide = torch.randn((M, c["K"] + c["spare"]), device=DEV, generator=gen)
        wide *= torch.empty((M, 1), device=DEV).uniform_(0.2, 5.0, generator=gen)  # tokens differ in size
        return {"x": wide.to(DTYPES[c["dtype"]])[:, :c["K"]]}
    if c["op"] == "gemm":
        return {"q": _i8(gen, M, c["K"]), "s": _scales(gen, M, around=0.03), "w": _i8(gen, c["R"], c["K"]),
                "ws": _scales(gen, c["R"], around=2e-3 / math.sqrt(c["K"])),
                "bias": torch.randn(c["R"], device=DEV, generator=gen) * 0.1 if c["bias"] else None}
    E, H, F, k = c["E"], c["H"], c["F"], c["k"]
    ids, w, n = _routing(gen, c)
    d = {"ids": ids, "n": n}
    if c["op"] == "up":
        # products near 1, where the SwiGLU bends
        d.update(q=_i8(gen, M, H), s=_scales(gen, M, around=0.03), gate=_i8(gen, E, F, H), up=_i8(gen, E, F, H),
                 gs=_scales(gen, E, F, around=0.03 / math.sqrt(H)), us=_scales(gen, E, F, around=0.03 / math.sqrt(H)),
                 h=torch.zeros((M * k, F), dtype=DTYPES[c["dtype"]], device=DEV))
    else:
        d.update(w=w, q=_i8(gen, M * k, F), s=_scales(gen, M * k, around=0.01), down=_i8(gen, E, H, F),
                 ds=_scales(gen, E, H, around=0.03 / math.sqrt(F)))
    return d


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    state = {"case": c, "in": d}
    if own:  # the weights' handles: pointers and sizes, no copy
        W = _package().I8Weights
        if c["op"] == "gemm":
            state["w"] = W(d["w"], d["ws"])
        elif c["op"] == "up":
            state["gate"], state["up"] = W(d["gate"], d["gs"]), W(d["up"], d["us"])
        elif c["op"] == "down":
            state["down"] = W(d["down"], d["ds"])
    return state


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    T, c, d = _package(), state["case"], state["in"]
    if c["op"] == "route":
        ids, w, n = T.route_scores(d["logits"], c["k"], bias=d["bias"], score=c["score"], n_group=c["groups"],
                                   topk_group=c["keep"], group_top=c["group_top"], renorm=c["renorm"],
                                   factor=c["factor"])
        return {"ids": ids[:, :c["k"]], "w": w[:, :c["k"]], "n": n}
    if c["op"] == "quant":
        q, s = T.quantize_rows(d["x"])
        return {"q": q, "scale": s}
    if c["op"] == "gemm":
        return T.gemm_i8(state["w"], d["q"], d["s"], bias=d["bias"], dtype=DTYPES[c["dtype"]])
    plan = T.experts_plan(d["ids"], d["n"], c["k"], c["E"])
    if c["op"] == "up":
        return T.experts_up_i8(state["gate"], state["up"], d["q"], d["s"], d["ids"], d["n"], c["k"], plan=plan,
                               out=d["h"])
    return T.experts_down_i8(state["down"], d["q"], d["s"], d["ids"], d["w"], d["n"], c["k"], plan=plan,
                             dtype=DTYPES[c["dtype"]])


def _run_plain(state):
    c, d = state["case"], state["in"]
    if c["op"] == "route":
        return _route_plain(c, d["logits"], d["bias"])
    if c["op"] == "quant":
        x = d["x"].float()
        top = x.abs().amax(1)
        kept = top >= 127 * 2.0 ** -126  # a smaller row has no normal scale: zero
        scale = torch.where(kept, torch.div(top, torch.full_like(top, 127.0)), torch.zeros_like(top))
        q = torch.round(x.double() * 127.0 / top.double()[:, None])  # 64 bits: values next to a border
        return {"q": torch.where(kept[:, None], q, torch.zeros_like(q)).to(torch.int8), "scale": scale}
    if c["op"] == "gemm":
        y = (d["q"].float() @ d["w"].float().T) * (d["s"][:, None] * d["ws"])
        return (y if d["bias"] is None else y + d["bias"]).to(DTYPES[c["dtype"]])
    k = c["k"]
    ids = d["ids"][:, :k]
    taken = torch.arange(k, device=DEV) < d["n"][:, None]  # [M][k]
    if c["op"] == "up":
        x = d["q"].float().repeat_interleave(k, 0)
        s = d["s"].repeat_interleave(k)[:, None]
        g, u = _products(ids, c["E"], [(x, d["gate"]), (x, d["up"])])
        expert = ids.reshape(-1).long()
        g, u = g * (s * d["gs"][expert]), u * (s * d["us"][expert])
        h = g / (1 + torch.exp(-g)) * u
        return torch.where(taken.reshape(-1, 1), h, torch.zeros_like(h)).to(DTYPES[c["dtype"]])
    y, = _products(ids, c["E"], [(d["q"].float(), d["down"])])
    y = y * (d["s"][:, None] * d["ds"][ids.reshape(-1).long()])
    w = torch.where(taken, d["w"][:, :k], torch.zeros_like(d["w"][:, :k]))
    return (y.view(c["M"], k, -1) * w[:, :, None]).sum(1).to(DTYPES[c["dtype"]])


def _route_plain(c, logits, bias):
    """Scores, choice and weights in 64 bits: the choice is between values that may be next to each other."""
    M, E, k = c["M"], c["E"], c["k"]
    l = logits.double()
    free = l > -math.inf
    none = torch.full_like(l, -math.inf)
    if c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(1, keepdim=True))
        s = e / e.sum(1, keepdim=True)
    key = torch.where(free, l if bias is None else s + bias.double(), none)
    if c["groups"] > 1:
        of = key if c["group_top"] == 1 else torch.where(free, s if bias is None else s + bias.double(), none)
        best = of.view(M, c["groups"], -1).sort(dim=2, descending=True).values[:, :, :c["group_top"]]
        first = best[:, :, 0]
        best = torch.where(best == -math.inf, torch.zeros_like(best), best).sum(2)
        best = torch.where(first == -math.inf, first, best)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        kept = torch.zeros((M, c["groups"]), dtype=torch.bool, device=DEV).scatter_(1, order, True)
        key = torch.where(kept.repeat_interleave(E // c["groups"], 1), key, none)
    top, ids = key.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    chosen = top > -math.inf
    w = torch.where(chosen, s.gather(1, ids), torch.zeros_like(top))
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(2.0 ** -1000)
    return {"ids": torch.where(chosen, ids, torch.full_like(ids, -1)).int(), "w": (w * c["factor"]).float(),
            "n": chosen.sum(1).int()}


def _products(ids, E, pairs):
    """Row i of each x [n][K] times the matrix of its expert in w [E][R][K] -> [n][R], in 32 bits.  Few rows take a copy of their
    expert's matrix each; many are sorted by expert into tiles of TILE rows, each expert's last one ragged."""
    expert = ids.reshape(-1).long()
    n = expert.numel()
    if n <= 2 * TILE:
        return [(w[expert].float() @ x[:, :, None])[:, :, 0] for x, w in pairs]
    order = expert.sort(stable=True).indices
    count = torch.zeros(E, dtype=torch.long, device=DEV).scatter_add_(0, expert, torch.ones_like(expert))
    tiles = (count + TILE - 1) // TILE
    first_row, first_tile = count.cumsum(0) - count, tiles.cumsum(0) - tiles
    sorted_expert = expert[order]
    in_expert = torch.arange(n, device=DEV) - first_row[sorted_expert]
    place = torch.empty_like(expert)
    place[order] = first_tile[sorted_expert] * TILE + in_expert
    T = n // TILE + E  # no fewer than there can be
    of_tile = torch.searchsorted(tiles.cumsum(0), torch.arange(T, device=DEV), right=True).clamp_max(E - 1)
    got = []
    for x, w in pairs:
        xt = torch.zeros((T * TILE, x.shape[1]), device=DEV)
        xt[place] = x
        y = torch.bmm(xt.view(T, TILE, -1), w[of_tile].float().transpose(1, 2))
        got.append(y.view(T * TILE, -1)[place])
    return got


# ---- the definitions, in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "route":
        return _exact_route(c, d)
    if c["op"] == "quant":
        x = d["x"].double()
        peak = x.abs().max(1, keepdim=True).values
        step = peak / 127
        level = x / step  # to the nearest, even between two
        return {"q": torch.where(peak >= 127 * 2.0 ** -126, level, torch.zeros_like(level)).round().to(torch.int8),
                "scale": step[:, 0]}
    if c["op"] == "gemm":
        y = torch.mm(d["q"].double() * d["s"].double()[:, None], d["w"].double().t() * d["ws"].double()[None, :])
        return y if d["bias"] is None else y.add_(d["bias"].double())
    M, k = c["M"], c["k"]
    if c["op"] == "up":
        out = torch.zeros((M * k, c["F"]), dtype=torch.float64, device=DEV)
    else:
        out = torch.zeros((M, c["H"]), dtype=torch.float64, device=DEV)
    live = torch.arange(SLOTS, device=DEV)[None, :] < d["n"][:, None]
    for e in range(c["E"]):
        t, j = torch.nonzero(live & (d["ids"] == e), as_tuple=True)
        if t.numel() == 0:
            continue
        if c["op"] == "up":
            x = d["q"][t].double() * d["s"][t, None].double()
            g = x @ (d["gate"][e].double() * d["gs"][e, :, None].double()).t()
            u = x @ (d["up"][e].double() * d["us"][e, :, None].double()).t()
            out[t * k + j] = g * torch.sigmoid(g) * u
        else:
            x = d["q"][t * k + j].double() * (d["s"][t * k + j].double() * d["w"][t, j].double())[:, None]
            out.index_add_(0, t, x @ (d["down"][e].double() * d["ds"][e, :, None].double()).t())
    return out


def _exact_route(c, d):
    """One choice at a time: the best group left, then the best expert left, the lower index of equal ones."""
    M, E, k, G = c["M"], c["E"], c["k"], c["groups"]
    l = d["logits"].double()
    gone = torch.isinf(l)
    s = torch.sigmoid(l) if c["score"] == "sigmoid" else torch.softmax(l, 1)
    worth = s + d["bias"].double() if c["bias"] else s
    low = torch.finfo(torch.float64).min
    worth = worth.masked_fill(gone, low)
    if G > 1:
        two = worth.view(M, G, -1).topk(min(c["group_top"], E // G), 2).values
        sums = two.clamp_min(0).sum(2) if not c["bias"] else two.masked_fill(two == low, 0).sum(2)
        sums = sums.masked_fill(two[:, :, 0] == low, low)
        keep = torch.zeros((M, G), dtype=torch.bool, device=DEV)
        for _ in range(c["keep"]):
            at = sums.masked_fill(keep, -math.inf).max(1, keepdim=True).indices
            keep.scatter_(1, at, True)
        worth = worth.masked_fill(~keep[:, :, None].expand(M, G, E // G).reshape(M, E), low)
    ids, n = torch.full((M, k), -1, dtype=torch.int32, device=DEV), torch.zeros(M, dtype=torch.int32, device=DEV)
    w = torch.zeros((M, k), dtype=torch.float64, device=DEV)
    for j in range(k):
        top, at = worth.max(1, keepdim=True)
        there = top[:, 0] > low
        ids[:, j] = torch.where(there, at[:, 0].int(), ids[:, j])
        w[:, j] = torch.where(there, s.gather(1, at)[:, 0], w[:, j])
        n += there.int()
        worth = worth.scatter(1, at, low)
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, w)
    return {"ids": ids, "w": w * c["factor"], "n": n}


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    c = case
    M = c["M"]
    if c["op"] == "route":
        return {"bytes": 4 * M * c["E"] + 8 * M * c["k"] + 4 * M + (4 * c["E"] if c["bias"] else 0),
                "flops": 10 * M * c["E"]}
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "quant":
        return {"bytes": M * c["K"] * (size + 1) + 4 * M, "flops": 4 * M * c["K"]}
    if c["op"] == "gemm":
        R, K = c["R"], c["K"]
        return {"bytes": M * K + R * K + 4 * (M + R) + (4 * R if c["bias"] else 0) + size * M * R,
                "flops": 2 * M * R * K}
    E, H, F, k = c["E"], c["H"], c["F"], c["k"]
    share = [(e + 1) ** -c["skew"] for e in range(E)]
    mean = (k + 1) / 2 if c["ragged"] else k
    touched = sum(1 - (1 - min(1.0, mean * p / sum(share))) ** M for p in share)
    n = M * mean
    if c["op"] == "up":
        return {"bytes": touched * 2 * F * (H + 4) + M * (H + 4) + size * n * F + 4 * M * (k + 1),
                "flops": 4 * n * F * H}
    return {"bytes": touched * H * (F + 4) + n * (F + 4) + size * M * H + 4 * M * (2 * k + 1), "flops": 2 * n * F * H}
