"""Operators of a mixture-of-experts layer, as measurable cases: tokens sorted by expert and back with
their gradients, MXFP4 (microscaled 4-bit float) quantisation, products of MXFP4 matrices, and the whole
expert layer in MXFP4.

With `own` false, `run` computes them from elementary torch operations; with `own` true it makes the calls
that a program makes of the library. Shapes are the repository's own: hidden 2048 / expert width 512 (the
benchmark's layer), 2560 / 640 (the reference's model), 512 / 256 and 384 / 640 (the tests').

MXFP4: blocks of 32 values share a scale 2^e, e = max(floor(log2(largest magnitude)) - 2, -127), held as
the byte e + 127; an element is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, to nearest with ties to the
even code, beyond 6 the 6; two elements a byte, the earlier one in the low half.
"""
from __future__ import annotations

import math

import torch

own = False

SHAPES = ((2048, 512), (2560, 640), (512, 256), (384, 640))   # (hidden, expert width)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed() -> list[dict]:
    return [
        # one decoded token's activations on their way into an MXFP4 product, and the values that the codes stand for
        {"name": "quantize_token", "kind": "quantize", "T": 1, "n": 2048, "dtype": "f32"},
        # a long prompt's activations
        {"name": "quantize_prompt", "kind": "quantize", "T": 16384, "n": 2048, "dtype": "bf16"},
        # a dense layer's product for one token, an odd number of output rows
        {"name": "product_token", "kind": "product", "T": 1, "n": 2560, "rows": 1001, "E": 1, "K": 1, "out": "f32", "drop": 0.0},
        # one product of the expert layer for a short prompt, padded to a batch: a part of the slots belongs to nobody
        {"name": "product_experts", "kind": "product", "T": 1000, "n": 2560, "rows": 640, "E": 128, "K": 8, "out": "bf16", "drop": 0.06},
        # one user, plain decoding: a token through the expert layer; latency and launches count
        {"name": "layer_1", "kind": "layer", "T": 1, "n": 2048, "ff": 512, "E": 512, "K": 10, "dtype": "f32", "zipf": False, "drop": 0.0},
        # the largest decode batch
        {"name": "layer_64", "kind": "layer", "T": 64, "n": 2048, "ff": 512, "E": 512, "K": 10, "dtype": "f32", "zipf": False, "drop": 0.0},
        # a prompt chunk with skewed routing: few experts take most of the tokens, many take a handful
        {"name": "layer_4096", "kind": "layer", "T": 4096, "n": 2048, "ff": 512, "E": 512, "K": 10, "dtype": "bf16", "zipf": True, "drop": 0.0},
        # a long prompt, uniform routing: the largest case
        {"name": "layer_16384", "kind": "layer", "T": 16384, "n": 2048, "ff": 512, "E": 512, "K": 10, "dtype": "bf16", "zipf": False, "drop": 0.0},
        # a ragged decode batch around experts of the program's own: sort, and the weighted way back
        {"name": "sort_37", "kind": "sort", "T": 37, "n": 2560, "E": 512, "K": 10, "dtype": "f32", "zipf": False, "drop": 0.0},
        # a long prompt around experts of the program's own
        {"name": "sort_16384", "kind": "sort", "T": 16384, "n": 2048, "E": 512, "K": 10, "dtype": "bf16", "zipf": True, "drop": 0.0},
        # the backward pass of the same, a short odd sequence, down to the router's logits
        {"name": "grad_293", "kind": "grad", "T": 293, "n": 2560, "E": 128, "K": 8, "dtype": "f32", "zipf": False, "drop": 0.0},
        # a training step's sequences, with slots over an expert's capacity dropped
        {"name": "grad_4096", "kind": "grad", "T": 4096, "n": 2048, "E": 512, "K": 10, "dtype": "bf16", "zipf": True, "drop": 0.1},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng) -> dict:
    kind = rng.choice(("quantize", "product", "product", "layer", "layer", "sort", "grad"))
    n, ff = rng.choice(SHAPES)
    E, K = rng.choice((8, 64, 128, 512)), rng.choice((1, 2, 4, 6, 8, 10))
    K = min(K, E)
    drop = rng.choice((0.0, 0.0, 0.05, 0.3))
    if kind == "quantize":
        return {"kind": kind, "T": _log_int(rng, 1, 16384), "n": 32 * _log_int(rng, 1, 80), "dtype": rng.choice(tuple(DTYPES))}
    if kind == "product":
        if rng.random() < 0.4:
            return {"kind": kind, "T": _log_int(rng, 1, 4096), "n": 128 * _log_int(rng, 1, 20), "rows": _log_int(rng, 1, 2560), "E": 1, "K": 1,
                    "out": rng.choice(("f32", "bf16")), "drop": 0.0}
        return {"kind": kind, "T": _log_int(rng, 1, 4096), "n": n, "rows": rng.choice((ff, ff, _log_int(rng, 1, 1280))), "E": E, "K": K,
                "out": rng.choice(("f32", "bf16")), "drop": drop}
    if kind == "layer":
        return {"kind": kind, "T": _log_int(rng, 1, 8192), "n": n, "ff": ff, "E": E, "K": K, "dtype": rng.choice(tuple(DTYPES)), "zipf": rng.random() < 0.5,
                "drop": drop}
    n = rng.choice((n, n, _log_int(rng, 1, 2560)))
    return {"kind": kind, "T": _log_int(rng, 1, 16384 if kind == "sort" else 8192), "n": n, "E": E, "K": K, "dtype": rng.choice(tuple(DTYPES)),
            "zipf": rng.random() < 0.5, "drop": drop}


# ---- inputs -------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _normal(g, dtype: str, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda").to(DTYPES[dtype])


def _logits(g, T: int, E: int, zipf: bool) -> torch.Tensor:
    """Router logits [T][E]: N(0, 1), or a Zipf(1.1) law over the experts with Gumbel noise, whose largest K are K draws without repetition."""
    if not zipf:
        return torch.randn(T, E, generator=g, device=g.device)
    rank = torch.randperm(E, generator=g, device=g.device) + 1
    u = torch.rand(T, E, generator=g, device=g.device).clamp_(min=1e-7, max=1 - 1e-7)
    return -1.1 * rank.float().log() - (-u.log()).log()


def _routing(g, c):
    """ids int32 [T][K] (-1: the slot belongs to nobody), wts float [T][K]: softmax over the chosen logits, and the ids before any was dropped."""
    top = _logits(g, c["T"], c["E"], c.get("zipf", False)).topk(c["K"], dim=1)
    chosen, wts = top.indices.to(torch.int32).contiguous(), torch.softmax(top.values, 1)
    ids = chosen.clone()
    if c["drop"]:
        ids[torch.rand(ids.shape, generator=g, device=g.device) < c["drop"]] = -1
        if c["T"] > 4:
            ids[-(c["T"] // 5):][torch.rand(c["T"] // 5, generator=g, device=g.device) < 0.5] = -1   # padding: tokens with no slot at all
    return ids, wts.contiguous(), chosen


def _weights(g, E: int, rows: int, n: int):
    """E matrices [rows][n] of normal weights in MXFP4: codes [E][rows][n / 2], scales [E][rows][n / 32]. Pieces of 32 are taken
    from a pool of 2^16 quantized ones, a row's scales vary with the row."""
    pool_codes, pool_scales = _to_codes(torch.randn(1 << 16, 32, generator=g, device="cuda"))
    at = torch.randint(0, 1 << 16, (E * rows * (n // 32),), generator=g, device="cuda")
    scale_of = torch.randint(-7, -3, (E, rows, 1), generator=g, device="cuda")
    return pool_codes[at].view(E, rows, n // 2), (pool_scales[at].view(E, rows, n // 32).int() + scale_of).to(torch.uint8)


def prepare(case: dict, seed: int) -> dict:
    g, c = _gen(seed), case
    s = {"case": c}
    if c["kind"] == "quantize":
        spread = torch.exp2(torch.randint(-6, 7, (c["T"], c["n"] // 32, 1), generator=g, device="cuda").float())
        s["x"] = (torch.randn(c["T"], c["n"] // 32, 32, generator=g, device="cuda") * spread).view(c["T"], c["n"]).to(DTYPES[c["dtype"]])
        return s
    if c["kind"] == "product":
        s["xq"] = _to_codes(torch.randn(c["T"], c["n"], generator=g, device="cuda"))
        s["w"] = _weights(g, c["E"], c["rows"], c["n"])
        s["y"] = torch.zeros(c["T"] * c["K"], c["rows"], dtype=DTYPES[c["out"]], device="cuda")   # rows that belong to no expert stay as they are
        if c["E"] > 1:
            s["ids"], _, _ = _routing(g, c)
            s["plan"] = _sorted(s["ids"], c["E"])
        if own:
            from flashrt_b200 import mxfp4
            s["W"] = mxfp4.pack(*s["w"])   # the weights as the kernels read them: laid out once, when they are loaded
        return s
    s["ids"], s["wts"], s["chosen"] = _routing(g, c)
    if c["kind"] == "layer":
        s["x"] = _normal(g, c["dtype"], c["T"], c["n"])
        s["w"] = [_weights(g, c["E"], *shape) for shape in ((c["ff"], c["n"]), (c["ff"], c["n"]), (c["n"], c["ff"]))]
        if own:
            from flashrt_b200 import moe, mxfp4
            s["W"] = [mxfp4.pack(*w) for w in s["w"]]
            s["ws"] = moe.workspace(mxfp4.moe_layer_workspace_bytes(c["T"], c["K"], c["n"], c["ff"], c["E"]))
        return s
    S = c["T"] * c["K"]
    s["ys"] = _normal(g, c["dtype"], S, c["n"])
    if c["kind"] == "sort":
        s["x"] = _normal(g, c["dtype"], c["T"], c["n"])
        s["xs"] = torch.zeros(S, c["n"], dtype=DTYPES[c["dtype"]], device="cuda")   # rows behind the last expert's stay as they are
    else:
        s["gxs"], s["gout"] = _normal(g, c["dtype"], S, c["n"]), _normal(g, c["dtype"], c["T"], c["n"])
        s["row_of"] = _sorted(s["ids"], c["E"])[2]   # kept from the forward pass
        s["gys"] = torch.zeros(S, c["n"], dtype=DTYPES[c["dtype"]], device="cuda")
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _to_codes(x: torch.Tensor):
    """MXFP4 codes uint8 [T][n / 2] and scales uint8 [T][n / 32] of x [T][n]."""
    T, n = x.shape
    v = x.float().view(T, n // 32, 32)
    amax = v.abs().amax(2)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp_(min=-127)   # frexp: amax = m * 2^exponent, m in [0.5, 1)
    v = torch.ldexp(torch.ldexp(v, -(e // 2).unsqueeze(2)), -(e - e // 2).unsqueeze(2))   # x / 2^e, in two exact steps
    a = v.abs()
    code = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5).int()
    code = torch.where(v < 0, code + 8, code).view(T, n // 2, 2)
    return (code[..., 0] | code[..., 1] << 4).to(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values that the codes [..][n / 2] and scales [..][n / 32] stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).int()
    v = table[both].view(*scales.shape, 32)
    return torch.ldexp(v, (scales.int() - 127).unsqueeze(-1)).view(*codes.shape[:-1], codes.shape[-1] * 2)


def _sorted(ids: torch.Tensor, E: int):
    """offsets [E + 1], slot_of [S], row_of [T][K]: slots in the order of their experts, in slot order within one."""
    flat = ids.view(-1).long()
    key = torch.where(flat < 0, E, flat)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=E + 1)[:E]
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    place = torch.arange(flat.numel(), device=ids.device)
    live = place < offsets[-1]
    slot_of = torch.where(live, order, -1)
    row_of = torch.empty_like(order)
    row_of[order] = torch.where(live, place, -1)
    return offsets.int(), slot_of.int(), row_of.int().view_as(ids)


def _experts_product(xs, w, offsets, y):
    """y[r] = W_e xs[r] for the rows of each expert, one expert after the other."""
    at = offsets.tolist()
    for e, (a, b) in enumerate(zip(at, at[1:])):
        if b > a:
            y[a:b] = (xs[a:b] @ _values(w[0][e], w[1][e]).t()).to(y.dtype)
    return y


def _back(ys, wts, row_of):
    """sum over a token's slots of wts * ys[row], in 32 bits."""
    w = torch.where(row_of < 0, 0.0, wts).unsqueeze(2)
    picked = ys[row_of.clamp(min=0).long()].float()
    return (torch.where(w == 0, 0.0, picked) * w).sum(1)


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        return _values(*_to_codes(s["x"])).to(torch.float32 if c["dtype"] == "f32" else torch.bfloat16)
    if kind == "product":
        x = _values(*s["xq"])
        if c["E"] == 1:
            return (x @ _values(s["w"][0][0], s["w"][1][0]).t()).to(DTYPES[c["out"]])
        offsets, slot_of, _ = s["plan"]
        return _experts_product(x[slot_of.clamp(min=0).long() // c["K"]], s["w"], offsets, s["y"])
    if kind == "layer":
        offsets, slot_of, row_of = _sorted(s["ids"], c["E"])
        xs = _values(*_to_codes(s["x"]))[slot_of.clamp(min=0).long() // c["K"]]
        rows = torch.zeros(2, xs.shape[0], c["ff"], device="cuda")
        g, u = (_experts_product(xs, w, offsets, r) for w, r in zip(s["w"], rows))
        h = _values(*_to_codes(g / (1 + torch.exp(-g)) * u))
        ys = _experts_product(h, s["w"][2], offsets, torch.zeros(xs.shape[0], c["n"], device="cuda"))
        return _back(ys, s["wts"], row_of).to(torch.bfloat16)
    if kind == "sort":
        offsets, slot_of, row_of = _sorted(s["ids"], c["E"])
        live = row_of >= 0
        s["xs"][row_of[live].long()] = s["x"].unsqueeze(1).expand(-1, c["K"], -1)[live]
        return offsets, slot_of, row_of, s["xs"], _back(s["ys"], s["wts"], row_of).to(s["ys"].dtype)
    row_of, live = s["row_of"], s["row_of"] >= 0
    gx = _back(s["gxs"], torch.ones_like(s["wts"]), row_of).to(s["gxs"].dtype)
    s["gys"][row_of[live].long()] = (s["wts"].unsqueeze(2) * s["gout"].unsqueeze(1).float())[live].to(s["gys"].dtype)
    gw = (s["ys"][row_of.clamp(min=0).long()].float() * s["gout"].unsqueeze(1).float()).sum(2)
    gw = torch.where(live, gw, 0.0)
    gl = torch.zeros(c["T"], c["E"], device="cuda")
    inner = (s["wts"] * gw).sum(1, keepdim=True)
    gl.scatter_add_(1, s["chosen"].long(), s["wts"] * (gw - inner))   # a dropped slot's logit took part in the softmax
    return gx, s["gys"], gw, gl


# ---- the library's calls ------------------------------------------------------------------------

def _run_own(s):
    from flashrt_b200 import moe, mxfp4
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        return mxfp4.dequantize(*mxfp4.quantize(s["x"]), dtype=torch.float32 if c["dtype"] == "f32" else torch.bfloat16)
    if kind == "product":
        if c["E"] == 1:
            return mxfp4.matmul(*s["xq"], s["W"], out=s["y"])
        offsets, slot_of, _ = s["plan"]
        return mxfp4.moe_matmul(*s["xq"], s["W"], offsets, slot_of, c["K"], out=s["y"])
    if kind == "layer":
        return mxfp4.moe_layer(s["x"], s["ids"], s["wts"], *s["W"], dtype=torch.bfloat16, ws=s["ws"])
    if kind == "sort":
        offsets, slot_of, row_of = moe.moe_sort(s["ids"], c["E"])
        return offsets, slot_of, row_of, moe.moe_sort_rows(s["x"], row_of, out=s["xs"]), moe.moe_unsort_rows(s["ys"], s["wts"], row_of)
    gx = moe.moe_sort_rows_backward(s["gxs"], s["row_of"])
    gys, gw = moe.moe_unsort_rows_backward(s["gout"], s["ys"], s["wts"], s["row_of"], gys=s["gys"])
    return gx, gys, gw, moe.moe_route_topk_backward(gw, s["wts"], s["chosen"], c["E"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------

def _expected(c) -> tuple[float, float]:
    """Slots that belong to an expert, and experts with one at least, of a case's routing law (one sample of it)."""
    g = torch.Generator()
    g.manual_seed(1)
    ids, _, _ = _routing(g, c)
    ids = ids[ids >= 0]
    return float(ids.numel()), float(torch.unique(ids).numel())


def work(case: dict) -> dict:
    c = case
    n = c["n"]
    if c["kind"] == "quantize":   # x read, codes and scales written and read back, values written
        return {"bytes": c["T"] * n * (SIZE[c["dtype"]] + 2 * 17 / 32 + (4 if c["dtype"] == "f32" else 2)), "flops": 2 * c["T"] * n}
    live, experts = (c["T"], 1.0) if c["E"] == 1 else _expected(c)
    S, T, K, E = c["T"] * c["K"], c["T"], c["K"], c["E"]
    if c["kind"] == "product":
        return {"bytes": 17 / 32 * n * (experts * c["rows"] + T) + live * c["rows"] * SIZE[c["out"]], "flops": 2 * live * n * c["rows"]}
    if c["kind"] == "layer":
        return {"bytes": 17 / 32 * 3 * n * c["ff"] * experts + T * n * (SIZE[c["dtype"]] + 2) + 8 * S, "flops": 6 * live * n * c["ff"]}
    z = SIZE[c["dtype"]]
    if c["kind"] == "sort":   # ids and weights in, plan out; x in, its copies out; ys in, their sums out
        return {"bytes": 4 * (4 * S + E) + z * n * (2 * T + 2 * live), "flops": 2 * live * n}
    return {"bytes": 4 * (4 * S + T * E) + z * n * (2 * T + 3 * live), "flops": 4 * live * n}


# ---- from the definition, in 64 bits ------------------------------------------------------------

def _exact_values(x: torch.Tensor) -> torch.Tensor:
    """What x [T][n], in 64 bits, becomes in MXFP4."""
    v = x.double().view(x.shape[0], -1, 32)
    big = v.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(torch.where(big > 0, big, 1.0)))
    e = torch.where(torch.exp2(e) > big, e - 1, e)          # where the logarithm was rounded up to a whole number, or down
    e = torch.where(torch.exp2(e + 1) <= big, e + 1, e)
    unit = torch.exp2(torch.clamp(e - 2, min=-127))
    v = v / unit
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    a = v.abs().clamp(max=6)
    hi = torch.bucketize(a, grid).clamp(max=7)              # grid[hi - 1] < a <= grid[hi]
    lo = (hi - 1).clamp(min=0)
    below, above = a - grid[lo], grid[hi] - a
    pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (torch.where(v < 0, -grid[pick], grid[pick]) * unit).view(x.shape)


def _exact_decoded(codes, scales):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    nibbles = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.long, device=codes.device)
    nibbles[..., 0::2], nibbles[..., 1::2] = codes.long() % 16, codes.long() // 16
    sign = torch.where(nibbles > 7, -1.0, 1.0).double()
    return sign * table[nibbles % 8] * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def exact(case: dict, seed: int):
    s, c = prepare(case, seed), case
    kind = c["kind"]
    if kind == "quantize":
        return _exact_values(s["x"])
    if kind == "product" and c["E"] == 1:
        return _exact_decoded(*s["xq"]) @ _exact_decoded(s["w"][0][0], s["w"][1][0]).t()
    ids = s["ids"].long()
    T, K, E, n = c["T"], c["K"], c["E"], c["n"]
    flat = ids.reshape(-1)
    slots = torch.cat([(flat == e).nonzero()[:, 0] for e in range(E)])      # the slots, expert after expert
    where = torch.full((T * K,), -1, dtype=torch.long, device=ids.device)
    where[slots] = torch.arange(slots.numel(), device=ids.device)
    count = [int((flat == e).sum()) for e in range(E)]
    begin = [sum(count[:e]) for e in range(E + 1)]

    def per_expert(rows, w, width):
        y = torch.zeros(T * K, width, dtype=torch.float64, device=rows.device)
        for e in range(E):
            if count[e]:
                y[begin[e]:begin[e + 1]] = rows[begin[e]:begin[e + 1]] @ _exact_decoded(w[0][e], w[1][e]).T
        return y

    if kind == "product":
        return per_expert(_exact_decoded(*s["xq"])[slots // K], s["w"], c["rows"])
    out = torch.zeros(T, n, dtype=torch.float64, device=ids.device)
    if kind == "layer":
        xs = _exact_values(s["x"])[slots // K]
        g, u = per_expert(xs, s["w"][0], c["ff"]), per_expert(xs, s["w"][1], c["ff"])
        ys = per_expert(_exact_values(g * torch.sigmoid(g) * u), s["w"][2], n)
        return out.index_add_(0, slots // K, ys[:slots.numel()] * s["wts"].double().reshape(-1)[slots].unsqueeze(1))
    slot_of = torch.full((T * K,), -1, dtype=torch.long, device=ids.device)
    slot_of[:slots.numel()] = slots
    w = s["wts"].double().reshape(-1)[slots].unsqueeze(1)
    if kind == "sort":
        xs = torch.zeros(T * K, n, dtype=torch.float64, device=ids.device)
        xs[:slots.numel()] = s["x"].double()[slots // K]
        out.index_add_(0, slots // K, s["ys"][:slots.numel()].double() * w)
        return None, None, None, xs, out
    gx = out.index_add(0, slots // K, s["gxs"][:slots.numel()].double())
    rows = s["gout"].double()[slots // K]
    gys = torch.zeros(T * K, n, dtype=torch.float64, device=ids.device)
    gys[:slots.numel()] = rows * w
    gw = torch.zeros(T * K, dtype=torch.float64, device=ids.device)
    gw[slots] = (rows * s["ys"][:slots.numel()].double()).sum(1)
    gw = gw.view(T, K)
    p = s["wts"].double()
    gl = torch.zeros(T * E, dtype=torch.float64, device=ids.device)
    gl[(torch.arange(T, device=ids.device).unsqueeze(1) * E + s["chosen"].long()).view(-1)] = (p * gw - p * (p * gw).sum(1, keepdim=True)).view(-1)
    return gx, gys, gw, gl.view(T, E)
