"""Microscaled 4-bit products (values of 4 bits, a power of two for each 32 of them), dense and for a router's experts, and a
whole MoE layer on such experts for a few tokens: the calls that performance work on these operators is measured on.

A case names one operator and its sizes:

  quant   x [M][K] -> 4-bit rows and their scales (`quantize_mx4`), read back (`dequantize_mx4`)
  gemm    4-bit rows x a 4-bit matrix [R][K] -> [M][R] (`gemm_mx4`)
  up      each token through its k experts' gate and up products and SwiGLU -> [M * k][F] (`experts_plan`,
          `experts_up_mx4`)
  down    the activation rows through their experts' down products, weighted and summed per token -> [M][H]
          (`experts_plan`, `experts_down_mx4`)
  layer   x [M][H] through the router, the choice of k experts by scores, those experts and the shared ones -> [M][H]
          (`moe_mx4`): the experts' weights in 4 bits, everything else in 32

M tokens, E experts of width F, hidden size H.  dtype: of x in `quant` and `layer`, of the output in all but `quant`.
spare: values behind each row of x that belong to something else (a slice of a wider tensor).  skew: an expert's load
falls as 1 / (rank + 1)^skew.  ragged: a token takes 1 to k experts, as routing by mass gives them.

A 4-bit value is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; a block of 32 neighbours of a row shares a scale 2^e, kept as
the byte e + 127.  Packed: two values a byte, the first in the low half.  A row's last block is filled up with zeros.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
SLOTS = 32  # experts a row of ids and weights has room for
BLOCK = 32  # values that share a scale
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TILE = 64   # entries of one expert that the plain form multiplies together
PART = 1 << 26  # values that are quantised or read back at a time


def _package():
    """This repository's package, as a program has it imported once."""
    if "trmoe" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tr-infer_amd"))
        import trmoe  # noqa: F401
    return sys.modules["trmoe"]


# ---- the cases -------------------------------------------------------------------------------------

def _quant(M, K, dtype, spare=0, **more):
    return dict(more, op="quant", M=M, K=K, dtype=dtype, spare=spare)


def _gemm(M, R, K, dtype, bias=False, **more):
    return dict(more, op="gemm", M=M, R=R, K=K, dtype=dtype, bias=bias)


def _experts(op, M, k, E, H, F, dtype, skew=0.0, ragged=False, **more):
    return dict(more, op=op, M=M, k=k, E=E, H=H, F=F, dtype=dtype, skew=skew, ragged=ragged)


def _layer(M, k, E, H, F, dtype, score="sigmoid", bias=True, groups=1, keep=1, renorm=True, factor=1.0, shared=0,
           gated=False, **more):
    return dict(more, op="layer", M=M, k=k, E=E, H=H, F=F, dtype=dtype, score=score, bias=bias, groups=groups, keep=keep,
                renorm=renorm, factor=factor, shared=shared, gated=gated)


def listed():
    return [
        # the rows of a few decoded tokens
        _quant(4, 2048, "f32", name="mx4_quant_decode"),
        # the rows of a large prefill, a slice of a wider projection's output
        _quant(8192, 4096, "bf16", spare=1024, name="mx4_quant_prefill"),
        # a dense projection of one decoded token: the weights are read once
        _gemm(1, 12288, 2560, "f32", name="mx4_gemm_decode"),
        # a short prompt, nothing a multiple of anything
        _gemm(77, 5003, 1999, "f16", bias=True, name="mx4_gemm_ragged"),
        # the same projection as the first in a large prefill
        _gemm(4096, 12288, 2560, "bf16", name="mx4_gemm_prefill"),
        # four sequences' tokens through their ten experts each
        _experts("up", 4, 10, 512, 2048, 512, "f32", name="mx4_up_decode"),
        # a prompt on fewer, wider experts, unevenly loaded
        _experts("up", 2000, 8, 128, 2048, 768, "bf16", skew=0.5, name="mx4_up_prefill"),
        # a short prompt whose tokens take one to six experts, odd sizes
        _experts("down", 150, 6, 60, 1100, 347, "f16", skew=0.3, ragged=True, name="mx4_down_ragged"),
        # a large prefill
        _experts("down", 4096, 10, 512, 2048, 512, "f32", skew=0.3, name="mx4_down_prefill"),
        # one decoded token through the layer, router to sum: softmax over 512 experts, a shared one behind its own gate
        _layer(1, 10, 512, 2048, 512, "bf16", score="softmax", bias=False, shared=1, gated=True, name="mx4_layer_decode"),
        # eight sequences' tokens: sigmoid scores, a balance bias, 4 of 8 groups, a shared expert
        _layer(8, 8, 256, 2048, 768, "f32", groups=8, keep=4, factor=2.5, shared=1, name="mx4_layer_batch"),
        # three tokens on a small layer, nothing a multiple of anything
        _layer(3, 2, 10, 650, 215, "f16", score="softmax", bias=False, name="mx4_layer_small"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "up", "up", "down", "down", "layer", "layer"])
    if op == "quant":
        K = _log(rng, 32, 12288)
        return _quant(_log(rng, 1, min(8192, 8192 * 4096 // K)), K, rng.choice(list(DTYPES)),
                      spare=rng.choice([0, 0, 8, 96, 1]))
    if op == "gemm":
        R, K = _log(rng, 64, 16384), _log(rng, 64, 12288)
        return _gemm(_log(rng, 1, min(4096, 4096 * 12288 * 2560 // (R * K))), R, K, rng.choice(list(DTYPES)),
                     bias=rng.random() < 0.5)
    E, H, F = _log(rng, 4 if op == "layer" else 8, 512), _log(rng, 256, 2560), _log(rng, 64, 1024)
    while E * H * F > 512 * 2048 * 512:
        E //= 2
    if op == "layer":
        groups = rng.choice([1, 1, 2, 4])
        E = max(groups, E // groups * groups)
        keep = rng.randint(1, groups)
        shared = rng.choice([0, 0, 1, 2])
        return _layer(_log(rng, 1, 8), rng.randint(1, min(10, keep * (E // groups))), E, H, F, rng.choice(list(DTYPES)),
                      score=rng.choice(["sigmoid", "softmax"]), bias=rng.random() < 0.5, groups=groups, keep=keep,
                      renorm=rng.random() < 0.7, factor=rng.choice([1.0, 2.5]), shared=shared,
                      gated=shared > 0 and rng.random() < 0.5)
    k = rng.randint(1, min(10, E))
    M = _log(rng, 1, 4096)
    while M * k * H * F > 4096 * 10 * 2048 * 512:
        M = (M + 1) // 2
    return _experts(op, M, k, E, H, F, rng.choice(list(DTYPES)), skew=rng.choice([0.0, 0.3, 0.8]),
                    ragged=rng.random() < 0.3)


# ---- 4-bit values ----------------------------------------------------------------------------------

def _up(n, to):
    return (n + to - 1) // to * to


def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _split(x):
    """x [..][k] -> its values over their blocks' scales, in 64 bits, the scales' exponents [..][blocks], and which blocks
    hold only numbers.  The scale: the largest magnitude's power of two, over 4 (6 is the largest value)."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, _blocks(k) * BLOCK - k)).double()
    x = x.view(*x.shape[:-1], -1, BLOCK)
    top = x.abs().amax(-1)
    fine = top < math.inf  # NaN compares false
    e = torch.frexp(torch.where(fine & (top > 0), top, torch.full_like(top, 2.0 ** -200)))[1] - 1 - 2
    e = e.clamp(-127, 127)
    return torch.where(fine[..., None], x, torch.zeros_like(x)) * torch.exp2(-e.double())[..., None], e, fine


def _codes(v):
    """The codes of the 4-bit values nearest to v, ties to the even code, magnitudes above 6 to 6."""
    a = v.abs()
    c = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
         + (a > 5).int())
    return c + 8 * torch.signbit(v).int()


def _values(dtype):
    return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=DEV)


def _quantised(gen, *shape, sigma):
    """The 4-bit rows of normals of deviation sigma: packed, rows of whole blocks (16 bytes each), and the scales' bytes,
    rows a multiple of 4 bytes apart."""
    *lead, k = shape
    nb = _blocks(k)
    rows = math.prod(lead)
    q = torch.empty((rows, nb * BLOCK // 2), dtype=torch.uint8, device=DEV)
    s = torch.zeros((rows, _up(nb, 4)), dtype=torch.uint8, device=DEV)
    step = max(1, PART // k)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        v, e, _ = _split(torch.randn((n, k), device=DEV, generator=gen) * sigma)
        c = _codes(v).view(n, -1)
        q[at:at + n] = (c[:, 0::2] | c[:, 1::2] << 4).to(torch.uint8)
        s[at:at + n, :nb] = (e + 127).to(torch.uint8)
    return q.view(*lead, -1), s.view(*lead, -1)[..., :nb]


def _read(q, s, k, dtype=torch.float32):
    """The values that packed rows and scales stand for, [..][k]."""
    table = _values(dtype)
    v = torch.stack((table[(q & 15).long()], table[(q >> 4).long()]), -1).view(*q.shape[:-1], -1, BLOCK)
    v = v * torch.exp2(s.to(dtype) - 127)[..., None]
    return v.view(*q.shape[:-1], -1)[..., :k]


# ---- inputs ----------------------------------------------------------------------------------------

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
    if c["op"] == "quant":
        wide = torch.randn((M, c["K"] + c["spare"]), device=DEV, generator=gen)
        wide *= torch.empty((M, 1), device=DEV).uniform_(0.2, 5.0, generator=gen)  # tokens differ in size
        return {"x": wide.to(DTYPES[c["dtype"]])[:, :c["K"]]}
    if c["op"] == "gemm":
        R, K = c["R"], c["K"]
        return {"x": _quantised(gen, M, K, sigma=1.0), "w": _quantised(gen, R, K, sigma=1 / math.sqrt(K)),
                "bias": torch.randn(R, device=DEV, generator=gen) * 0.1 if c["bias"] else None}
    E, H, F, k = c["E"], c["H"], c["F"], c["k"]
    if c["op"] == "layer":
        n = E + c["shared"]
        return {"x": torch.randn((M, H), device=DEV, generator=gen).to(DTYPES[c["dtype"]]),
                "router": torch.randn((E, H), device=DEV, generator=gen) * (1.3 / math.sqrt(H)),
                "bias": torch.randn(E, device=DEV, generator=gen) * 0.05 if c["bias"] else None,
                "shared_gate": torch.randn(H, device=DEV, generator=gen) / math.sqrt(H) if c["gated"] else None,
                "gate": _quantised(gen, n, F, H, sigma=1 / math.sqrt(H)),
                "up": _quantised(gen, n, F, H, sigma=1 / math.sqrt(H)),
                "down": _quantised(gen, n, H, F, sigma=1 / math.sqrt(F))}
    ids, w, n = _routing(gen, c)
    d = {"ids": ids, "n": n}
    if c["op"] == "up":
        d.update(x=_quantised(gen, M, H, sigma=1.0), gate=_quantised(gen, E, F, H, sigma=1 / math.sqrt(H)),
                 up=_quantised(gen, E, F, H, sigma=1 / math.sqrt(H)),
                 h=torch.zeros((M * k, F), dtype=DTYPES[c["dtype"]], device=DEV))
    else:
        d.update(w=w, x=_quantised(gen, M * k, F, sigma=0.5), down=_quantised(gen, E, H, F, sigma=1 / math.sqrt(F)))
    return d


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    state = {"case": c, "in": d}
    if own:  # the weights' handles: pointers and sizes, no copy
        T = _package()
        if c["op"] == "gemm":
            state["w"] = T.MX4Weights(*d["w"], c["K"])
        elif c["op"] == "up":
            state["gate"], state["up"] = T.MX4Weights(*d["gate"], c["H"]), T.MX4Weights(*d["up"], c["H"])
        elif c["op"] == "down":
            state["down"] = T.MX4Weights(*d["down"], c["F"])
        elif c["op"] == "layer":
            state["layer"] = T.MX4Layer(T.MX4Weights(*d["gate"], c["H"]), T.MX4Weights(*d["up"], c["H"]),
                                        T.MX4Weights(*d["down"], c["F"]), router=d["router"], bias=d["bias"],
                                        n_shared=c["shared"], shared_gate=d["shared_gate"])
    return state


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    T, c, d = _package(), state["case"], state["in"]
    if c["op"] == "quant":
        q, s = T.quantize_mx4(d["x"])
        return T.dequantize_mx4(q, s, c["K"], dtype=d["x"].dtype)
    if c["op"] == "layer":
        return T.moe_mx4(state["layer"], d["x"], c["k"], score=c["score"], n_group=c["groups"], topk_group=c["keep"],
                         renorm=c["renorm"], factor=c["factor"])
    q, s = d["x"]
    if c["op"] == "gemm":
        return T.gemm_mx4(state["w"], q, s, bias=d["bias"], dtype=DTYPES[c["dtype"]])
    plan = T.experts_plan(d["ids"], d["n"], c["k"], c["E"])
    if c["op"] == "up":
        return T.experts_up_mx4(state["gate"], state["up"], q, s, d["ids"], d["n"], c["k"], plan=plan, out=d["h"])
    return T.experts_down_mx4(state["down"], q, s, d["ids"], d["w"], d["n"], c["k"], plan=plan, dtype=DTYPES[c["dtype"]])


def _run_plain(state):
    c, d = state["case"], state["in"]
    if c["op"] == "quant":
        v, e, fine = _split(d["x"])  # 64 bits: values next to a border
        y = _values(torch.float32)[_codes(v).long()] * torch.exp2(e.float())[..., None]
        y = torch.where(fine[..., None], y, torch.full_like(y, math.nan))
        return y.view(c["M"], -1)[:, :c["K"]].to(d["x"].dtype)
    if c["op"] == "gemm":
        y = _read(*d["x"], c["K"]) @ _read(*d["w"], c["K"]).T
        return (y if d["bias"] is None else y + d["bias"]).to(DTYPES[c["dtype"]])
    k = c["k"]
    if c["op"] == "layer":
        return _layer_plain(c, d)
    ids = d["ids"][:, :k]
    taken = torch.arange(k, device=DEV) < d["n"][:, None]  # [M][k]
    if c["op"] == "up":
        x = _read(*d["x"], c["H"]).repeat_interleave(k, 0)
        g, u = _products(ids, c["E"], c["H"], [(x, d["gate"]), (x, d["up"])])
        h = g / (1 + torch.exp(-g)) * u
        return torch.where(taken.reshape(-1, 1), h, torch.zeros_like(h)).to(DTYPES[c["dtype"]])
    y, = _products(ids, c["E"], c["F"], [(_read(*d["x"], c["F"]), d["down"])])
    w = torch.where(taken, d["w"][:, :k], torch.zeros_like(d["w"][:, :k]))
    return (y.view(c["M"], k, -1) * w[:, :, None]).sum(1).to(DTYPES[c["dtype"]])


def _layer_plain(c, d):
    """The choice in 64 bits, for it is between values that may be next to each other; the experts in 32."""
    M, E, k = c["M"], c["E"], c["k"]
    x64 = d["x"].double()
    l = x64 @ d["router"].double().T
    if c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(1, keepdim=True))
        s = e / e.sum(1, keepdim=True)
    key = l if d["bias"] is None else s + d["bias"].double()
    if c["groups"] > 1:
        of = (s if d["bias"] is None else key).view(M, c["groups"], -1)
        best = of.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        kept = torch.zeros((M, c["groups"]), dtype=torch.bool, device=DEV).scatter_(1, order, True)
        key = torch.where(kept.repeat_interleave(E // c["groups"], 1), key, torch.full_like(key, -math.inf))
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * c["factor"]
    if c["shared"]:
        ids = torch.cat((ids, torch.arange(E, E + c["shared"], device=DEV).expand(M, -1)), 1)
        g = torch.ones(M, dtype=torch.float64, device=DEV)
        if c["gated"]:
            g = 1 / (1 + torch.exp(-(x64 @ d["shared_gate"].double())))
        w = torch.cat((w, g[:, None].expand(-1, c["shared"])), 1)
    n = ids.shape[1]
    x = d["x"].float().repeat_interleave(n, 0)
    g, u = _products(ids, E + c["shared"], c["H"], [(x, d["gate"]), (x, d["up"])])
    h = g / (1 + torch.exp(-g)) * u
    y, = _products(ids, E + c["shared"], c["F"], [(h, d["down"])])
    return (y.view(M, n, -1) * w.float()[:, :, None]).sum(1).to(d["x"].dtype)


def _products(ids, E, K, pairs):
    """Row i of each x [n][K] times the matrix of its expert -> [n][R], in 32 bits.  Few rows take a copy of their expert's
    matrix each; many are sorted by expert into tiles of TILE rows, each expert's last one ragged."""
    expert = ids.reshape(-1).long()
    n = expert.numel()
    if n <= 2 * TILE:
        return [(_read(q[expert], s[expert], K) @ x[:, :, None])[:, :, 0] for x, (q, s) in pairs]
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
    for x, (q, s) in pairs:
        xt = torch.zeros((T * TILE, K), device=DEV)
        xt[place] = x
        w = _read(q, s, K)
        y = torch.bmm(xt.view(T, TILE, -1), w.transpose(1, 2).contiguous()[of_tile])
        got.append(y.view(T * TILE, -1)[place])
    return got


# ---- the definitions, in 64 bits -------------------------------------------------------------------

def _matrix(q, s, k):
    """Packed rows [rows][bytes] as numbers in 64 bits: sign, exponent and fraction of each code taken apart."""
    c = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.float64, device=DEV)
    for half in (0, 1):
        code = (q >> (4 * half)) & 15
        ex, frac, neg = ((code >> 1) & 3).double(), (code & 1).double(), (code >> 3).double()
        v = torch.where(ex == 0, frac / 2, (1 + frac / 2) * torch.pow(2.0, ex - 1))
        c[:, half::2] = v * (1 - 2 * neg)
    scale = torch.pow(2.0, s.double() - 127)
    return (c * scale.repeat_interleave(BLOCK, 1))[:, :k]


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "quant":
        return _exact_quant(c, d["x"].double())
    if c["op"] == "gemm":
        y = torch.mm(_matrix(*d["x"], c["K"]), _matrix(*d["w"], c["K"]).t())
        return y if d["bias"] is None else y.add_(d["bias"].double())
    if c["op"] == "layer":
        return _exact_layer(c, d)
    M, k = c["M"], c["k"]
    x = _matrix(*d["x"], c["H"] if c["op"] == "up" else c["F"])
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
            g = x[t] @ _matrix(d["gate"][0][e], d["gate"][1][e], c["H"]).t()
            u = x[t] @ _matrix(d["up"][0][e], d["up"][1][e], c["H"]).t()
            out[t * k + j] = g * torch.sigmoid(g) * u
        else:
            y = x[t * k + j] @ _matrix(d["down"][0][e], d["down"][1][e], c["F"]).t()
            out.index_add_(0, t, y * d["w"][t, j, None].double())
    return out


def _exact_quant(c, x):
    """Each value against every 4-bit value of its block's scale: the nearest, the even code of two."""
    M, K = x.shape
    out = torch.empty((M, K), dtype=torch.float64, device=DEV)
    table = _values(torch.float64)[:8]
    even = torch.arange(8, device=DEV) % 2 * 1e-9  # the odd code of two that are as near counts as a little further
    for at in range(0, K, BLOCK):
        b = x[:, at:at + BLOCK]
        top = b.abs().max(1, keepdim=True).values
        scale = torch.pow(2.0, torch.floor(torch.log2(top.clamp_min(2.0 ** -140))).clamp_min(-125) - 2)
        far = ((b.abs() / scale)[:, :, None] - table).abs() + even
        out[:, at:at + BLOCK] = table[far.argmin(2)] * scale * torch.sign(b)
    return out


def _exact_layer(c, d):
    """Token by token, one choice at a time, each expert's matrices by themselves."""
    M, E, k, G = c["M"], c["E"], c["k"], c["groups"]
    x = d["x"].double()
    out = torch.zeros((M, c["H"]), dtype=torch.float64, device=DEV)
    for t in range(M):
        l = d["router"].double() @ x[t]
        s = torch.sigmoid(l) if c["score"] == "sigmoid" else torch.softmax(l, 0)
        worth = s + d["bias"].double() if c["bias"] else s
        if G > 1:
            sums = worth.view(G, -1).topk(min(2, E // G), 1).values.sum(1)
            kept = torch.zeros(G, dtype=torch.bool, device=DEV)
            kept[sums.topk(c["keep"]).indices] = True
            worth = worth.masked_fill(~kept.repeat_interleave(E // G), -math.inf)
        chosen = worth.topk(k).indices
        w = s[chosen]
        w = (w / w.sum() if c["renorm"] else w) * c["factor"]
        took = list(zip(chosen.tolist(), w.tolist()))
        gate = torch.sigmoid(x[t] @ d["shared_gate"].double()).item() if c["gated"] else 1.0
        took += [(E + i, gate) for i in range(c["shared"])]
        for e, share in took:
            g = _matrix(d["gate"][0][e], d["gate"][1][e], c["H"]) @ x[t]
            u = _matrix(d["up"][0][e], d["up"][1][e], c["H"]) @ x[t]
            out[t] += share * (_matrix(d["down"][0][e], d["down"][1][e], c["F"]) @ (g * torch.sigmoid(g) * u))
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    c = case
    M = c["M"]
    size = 4 if c["dtype"] == "f32" else 2

    def row(k):  # a 4-bit row with its scales
        return _blocks(k) * (BLOCK // 2 + 1)

    if c["op"] == "quant":
        return {"bytes": 2 * M * c["K"] * size + 2 * M * row(c["K"]), "flops": 6 * M * c["K"]}
    if c["op"] == "gemm":
        R, K = c["R"], c["K"]
        return {"bytes": (M + R) * row(K) + (4 * R if c["bias"] else 0) + size * M * R, "flops": 2 * M * R * K}
    E, H, F, k = c["E"], c["H"], c["F"], c["k"]
    if c["op"] == "layer":
        touched = E * (1 - (1 - k / E) ** M) + c["shared"]
        n = M * (k + c["shared"])
        return {"bytes": 4 * E * H + touched * (2 * F * row(H) + H * row(F)) + 2 * size * M * H,
                "flops": 2 * M * E * H + 6 * n * F * H}
    share = [(e + 1) ** -c["skew"] for e in range(E)]
    mean = (k + 1) / 2 if c["ragged"] else k
    touched = sum(1 - (1 - min(1.0, mean * p / sum(share))) ** M for p in share)
    n = M * mean
    if c["op"] == "up":
        return {"bytes": touched * 2 * F * row(H) + M * row(H) + size * n * F + 4 * M * (k + 1), "flops": 4 * n * F * H}
    return {"bytes": touched * H * row(F) + n * row(F) + size * M * H + 4 * M * (2 * k + 1), "flops": 2 * n * F * H}
