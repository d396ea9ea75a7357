"""Operators around experts and projections in 16 bits, as measurable cases: products of sorted rows with their experts' matrices and both
gradients, SwiGLU rows kept in 8 bits for the backward pass, and low-rank adapters of many requests beside a shared projection.

With `own` false, `run` computes them from elementary torch operations; with `own` true it makes the calls that a program makes of the
library. Shapes are the repository's own: hidden 2048 / expert width 512 (the benchmark's layer), 2560 / 640 (the reference's model), 512 / 256
and 384 / 640 (the tests'); gate and up of an expert are one matrix of twice its width.

MXINT8: blocks of 32 values share a scale 2^e, e = max(floor(log2(largest magnitude)), -127), held as the byte e + 127; an element is an
8-bit integer, the value / 2^(e - 6) to nearest with ties to even, at most 127 in magnitude.
"""
from __future__ import annotations

import math
import random

import torch

own = False

SHAPES = ((2048, 512), (2560, 640), (512, 256), (384, 640))   # (hidden, expert width)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed() -> list[dict]:
    return [
        # one user, plain decoding: a token's rows through gate and up of its ten experts
        {"name": "product_1", "kind": "product", "T": 1, "n": 2048, "rows": 1024, "E": 512, "K": 10, "dtype": "bf16", "out": "bf16", "zipf": False, "drop": 0.0},
        # the largest decode batch: most experts have a row or two
        {"name": "product_64", "kind": "product", "T": 64, "n": 2048, "rows": 1024, "E": 512, "K": 10, "dtype": "bf16", "out": "f32", "zipf": False, "drop": 0.0},
        # a short prompt padded to a batch: a part of the slots belongs to nobody, experts have some sixty rows
        {"name": "product_1000", "kind": "product", "T": 1000, "n": 2560, "rows": 1280, "E": 128, "K": 8, "dtype": "f16", "out": "f16", "zipf": False, "drop": 0.06},
        # a long prompt, or the forward pass of a training step, with skewed routing: the largest case
        {"name": "product_16384", "kind": "product", "T": 16384, "n": 2048, "rows": 1024, "E": 128, "K": 8, "dtype": "bf16", "out": "bf16", "zipf": True, "drop": 0.0},
        # the backward pass of a short odd sequence: gradients of the rows, and of all matrices in 32 bits
        {"name": "grad_293", "kind": "grad", "T": 293, "n": 2560, "rows": 1280, "E": 128, "K": 8, "dtype": "f16", "out": "f32", "zipf": False, "drop": 0.05},
        # the backward pass of a training step
        {"name": "grad_8192", "kind": "grad", "T": 8192, "n": 2048, "rows": 1024, "E": 64, "K": 8, "dtype": "bf16", "out": "bf16", "zipf": False, "drop": 0.0},
        # what a short odd sequence keeps for its backward pass: tokens' rows, and gate and up rows, in 8 bits
        {"name": "kept_293", "kind": "kept", "T": 293, "n": 2560, "ff": 640, "K": 8, "dtype": "f32"},
        # and a training step's
        {"name": "kept_8192", "kind": "kept", "T": 8192, "n": 2048, "ff": 512, "K": 10, "dtype": "bf16"},
        # one user with an adapter, plain decoding: latency
        {"name": "adapter_1", "kind": "adapter", "T": 1, "R": 1, "L": 8, "rank": 16, "n": 2048, "rows": 2048, "dtype": "bf16", "out": "bf16", "none": 0.0},
        # a decode batch of as many users, each with an adapter of its own or none
        {"name": "adapter_64", "kind": "adapter", "T": 64, "R": 64, "L": 100, "rank": 16, "n": 2560, "rows": 2560, "dtype": "f16", "out": "f16", "none": 0.1},
        # decoding users and prompts in one batch, outputs in 32 bits
        {"name": "adapter_1000", "kind": "adapter", "T": 1000, "R": 41, "L": 100, "rank": 64, "n": 2048, "rows": 2560, "dtype": "bf16", "out": "f32", "none": 0.2},
        # a batch of long prompts
        {"name": "adapter_16384", "kind": "adapter", "T": 16384, "R": 24, "L": 16, "rank": 32, "n": 2048, "rows": 2048, "dtype": "bf16", "out": "bf16", "none": 0.1},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng) -> dict:
    kind = rng.choice(("product", "product", "grad", "kept", "adapter", "adapter"))
    n, ff = rng.choice(SHAPES)
    dtype = rng.choice(("bf16", "f16"))
    if kind == "kept":
        if rng.random() < 0.4:
            n, ff = 32 * _log_int(rng, 1, 80), 32 * _log_int(rng, 1, 32)
        return {"kind": kind, "T": _log_int(rng, 1, 8192), "n": n, "ff": ff, "K": rng.choice((1, 2, 4, 6, 8)), "dtype": rng.choice(tuple(DTYPES))}
    if kind == "adapter":
        T = _log_int(rng, 1, 16384)
        R = _log_int(rng, 1, min(T, 256))
        if T <= 256 and rng.random() < 0.5:
            R = T
        return {"kind": kind, "T": T, "R": R, "L": _log_int(rng, 1, 100), "rank": rng.choice((8, 16, 16, 24, 32, 64)),
                "n": rng.choice((n, n, 8 * _log_int(rng, 1, 256))), "rows": rng.choice((n, 2 * ff, _log_int(rng, 1, 2048))), "dtype": dtype,
                "out": rng.choice((dtype, dtype, "f32")), "none": rng.choice((0.0, 0.1, 0.5))}
    E, K = rng.choice((8, 64, 128)), rng.choice((1, 2, 4, 6, 8))
    drop, zipf, out = rng.choice((0.0, 0.0, 0.05, 0.3)), rng.random() < 0.5, rng.choice((dtype, dtype, "f32"))
    if kind == "product":
        rows = rng.choice((2 * ff, n, _log_int(rng, 1, 1280)))
        return {"kind": kind, "T": _log_int(rng, 1, 8192), "n": n, "rows": rows, "E": E, "K": K, "dtype": dtype, "out": out, "zipf": zipf, "drop": drop}
    return {"kind": kind, "T": _log_int(rng, 1, 4096), "n": n, "rows": rng.choice((2 * ff, 2 * ff, 8 * _log_int(rng, 1, 160))), "E": min(E, 64), "K": K,
            "dtype": dtype, "out": out, "zipf": zipf, "drop": drop}


# ---- inputs -------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6151 + 41)
    return g


def _normal(g, dtype: str, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda", dtype=DTYPES[dtype])


def _ids(g, c):
    """The experts of every slot, int32 [T][K], -1 where the slot belongs to nobody: the largest K of N(0, 1) logits, or K draws without repetition of a
    Zipf(1.1) law over the experts."""
    T, E, K = c["T"], c["E"], c["K"]
    if c["zipf"]:
        rank = torch.randperm(E, generator=g, device=g.device) + 1
        u = torch.rand(T, E, generator=g, device=g.device).clamp_(min=1e-7, max=1 - 1e-7)
        logits = -1.1 * rank.float().log() - (-u.log()).log()
    else:
        logits = torch.randn(T, E, generator=g, device=g.device)
    ids = logits.topk(K, dim=1).indices.to(torch.int32)
    if c["drop"]:
        ids[torch.rand(T, K, generator=g, device=g.device) < c["drop"]] = -1
        if T > 4:
            ids[T - T // 5:][torch.rand(T // 5, generator=g, device=g.device) < 0.5] = -1   # padding: tokens with no slot at all
    return ids


def _offsets(ids: torch.Tensor, E: int) -> torch.Tensor:
    """Where every expert's rows begin in the sorted order, and behind them where nobody's do: int32 [E + 1]."""
    flat = ids.view(-1).long()
    counts = torch.bincount(torch.where(flat < 0, E, flat), minlength=E + 1)[:E]
    return torch.cat((counts.new_zeros(1), counts.cumsum(0))).int()


def _requests(c, seed: int):
    """Token ranges and adapters of R requests: most have one token (they are decoding), every eighth is a prompt. Lists of R + 1 and R."""
    rng = random.Random(seed * 31 + 7)
    T, R = c["T"], c["R"]
    lengths = [1] * R
    prompts = rng.sample(range(R), max(1, R // 8))
    cuts = sorted(rng.randint(0, T - R) for _ in prompts[1:])
    for i, a, b in zip(prompts, [0] + cuts, cuts + [T - R]):
        lengths[i] += b - a
    offsets = [0]
    for m in lengths:
        offsets.append(offsets[-1] + m)
    return offsets, [-1 if rng.random() < c["none"] else rng.randrange(c["L"]) for _ in range(R)]


def prepare(case: dict, seed: int) -> dict:
    g, c = _gen(seed), case
    s = {"case": c}
    if c["kind"] == "kept":
        S, n, ff, dtype = c["T"] * c["K"], c["n"], c["ff"], c["dtype"]
        spread = torch.exp2(torch.randint(-4, 5, (c["T"], 1), generator=g, device="cuda").float())   # tokens of different magnitudes
        s["x"] = (torch.randn(c["T"], n, generator=g, device="cuda") * spread).to(DTYPES[dtype])
        s["gu"] = _normal(g, dtype, S, 2 * ff) * 1.5
        s["gh"] = _normal(g, dtype, S, ff)
        return s
    if c["kind"] == "adapter":
        T, n, rows, L, rank, dtype = c["T"], c["n"], c["rows"], c["L"], c["rank"], c["dtype"]
        s["requests"] = _requests(c, seed)
        offsets, which = s["requests"]
        s["offsets"], s["which"] = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (offsets, which))
        s["x"], s["y"] = _normal(g, dtype, T, n), _normal(g, c["out"], T, rows)   # the shared projection's outputs
        s["a"], s["b"] = _normal(g, dtype, L, rank, n) / math.sqrt(n), _normal(g, dtype, L, rows, rank) / math.sqrt(rank)
        s["scale"] = torch.exp2(torch.randint(-2, 2, (L,), generator=g, device="cuda").float())
        s["out"] = torch.zeros_like(s["y"])
        return s
    T, n, rows, E, K, dtype = c["T"], c["n"], c["rows"], c["E"], c["K"], c["dtype"]
    S = T * K
    s["offsets"] = _offsets(_ids(g, c), E)
    s["x"] = _normal(g, dtype, S, n)                            # sorted by expert
    s["w"] = _normal(g, dtype, E, rows, n).mul_(1 / math.sqrt(n))
    if c["kind"] == "product":
        s["y"] = torch.zeros(S, rows, dtype=DTYPES[c["out"]], device="cuda")   # rows that belong to no expert stay as they are
    else:
        s["gy"] = _normal(g, dtype, S, rows)
        s["gx"] = torch.zeros(S, n, dtype=DTYPES[dtype], device="cuda")
        s["gw"] = torch.zeros(E, rows, n, dtype=DTYPES[c["out"]], device="cuda")
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _experts(offsets: torch.Tensor):
    at = offsets.tolist()
    return [(e, a, b) for e, (a, b) in enumerate(zip(at, at[1:]))]


def _kept(x: torch.Tensor) -> torch.Tensor:
    """The values that x [rows][n] becomes in MXINT8, in 32 bits."""
    v = x.float().view(x.shape[0], -1, 32)
    amax = v.abs().amax(2, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 1, -127).clamp_(min=-127) - 6
    half = e // 2   # 2^e in two exact steps
    q = torch.ldexp(torch.ldexp(v, -half), half - e).round_().clamp_(-127, 127)
    return torch.ldexp(torch.ldexp(q, half), e - half).view(x.shape)


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "product":
        for e, a, b in _experts(s["offsets"]):
            if b > a:
                s["y"][a:b] = (s["x"][a:b].float() @ s["w"][e].float().t()).to(s["y"].dtype)
        return s["y"]
    if c["kind"] == "grad":
        for e, a, b in _experts(s["offsets"]):
            gy = s["gy"][a:b].float()
            s["gx"][a:b] = (gy @ s["w"][e].float()).to(s["gx"].dtype)
            s["gw"][e] = (gy.t() @ s["x"][a:b].float()).to(s["gw"].dtype)
        return s["gx"], s["gw"]
    if c["kind"] == "kept":
        dtype, ff = s["gu"].dtype, c["ff"]
        gu, gh = s["gu"].float(), s["gh"].float()
        h = gu[:, :ff] / (1 + torch.exp(-gu[:, :ff])) * gu[:, ff:]
        kept = _kept(s["gu"])
        g, u = kept[:, :ff], kept[:, ff:]
        sig = 1 / (1 + torch.exp(-g))
        ggu = torch.cat((gh * u * sig * (1 + g * (1 - sig)), gh * g * sig), 1)
        return h.to(dtype), ggu.to(dtype), (g * sig * u).to(dtype), _kept(s["x"]).to(dtype)
    offsets, which = s["requests"]
    s["out"].copy_(s["y"])
    for a, b, j in zip(offsets, offsets[1:], which):
        if j >= 0:
            v = s["x"][a:b].float() @ s["a"][j].float().t() * s["scale"][j]
            s["out"][a:b] = (s["y"][a:b].float() + v @ s["b"][j].float().t()).to(s["out"].dtype)
    return s["out"]


# ---- the library's calls ------------------------------------------------------------------------

def _run_own(s):
    from flashrt_b200 import adapters, moe, mxint8
    c = s["case"]
    if c["kind"] == "product":
        return moe.moe_matmul(s["x"], s["w"], s["offsets"], out=s["y"])
    if c["kind"] == "grad":
        return (moe.moe_matmul_backward_x(s["gy"], s["w"], s["offsets"], out=s["gx"]),
                moe.moe_matmul_backward_w(s["gy"], s["x"], s["offsets"], out=s["gw"]))
    if c["kind"] == "kept":
        h, codes, scales = mxint8.swiglu(s["gu"])
        x_codes, x_scales = mxint8.quantize(s["x"])
        ggu, again = mxint8.swiglu_backward(s["gh"], codes, scales)
        return h, ggu, again, mxint8.dequantize(x_codes, x_scales, dtype=s["x"].dtype)
    return adapters.add(s["y"], s["x"], s["a"], s["b"], s["offsets"], s["which"], scale=s["scale"], out=s["out"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------

def _expected(c) -> tuple[float, float]:
    """Slots that belong to an expert, and experts with one at least, of a case's routing law (one sample of it)."""
    g = torch.Generator()
    g.manual_seed(1)
    ids = _ids(g, c)
    ids = ids[ids >= 0]
    return float(ids.numel()), float(torch.unique(ids).numel())


def work(case: dict) -> dict:
    c = case
    z, n = SIZE[c["dtype"]], c["n"]
    if c["kind"] == "kept":   # gate and up in, the hidden rows and 8 bits out; these and the gradient in, two gradients and the hidden rows out; a token's row in, out and back
        S, kept = c["T"] * c["K"], 33 / 32
        return {"bytes": S * c["ff"] * (7 * z + 4 * kept) + c["T"] * n * (2 * z + 2 * kept), "flops": 40 * S * c["ff"] + 8 * c["T"] * n}
    rows = c["rows"]
    if c["kind"] == "adapter":
        offsets, which = _requests(c, 1)
        live = sum(b - a for a, b, j in zip(offsets, offsets[1:], which) if j >= 0)
        distinct = len({j for j in which if j >= 0})
        return {"bytes": z * (live * n + distinct * c["rank"] * (n + rows)) + 2 * SIZE[c["out"]] * c["T"] * rows, "flops": 2 * live * c["rank"] * (n + rows)}
    live, experts = _expected(c)
    if c["kind"] == "product":
        return {"bytes": z * (experts * rows * n + live * n) + SIZE[c["out"]] * live * rows, "flops": 2 * live * n * rows}
    return {"bytes": z * (experts * rows * n + live * (2 * n + rows)) + SIZE[c["out"]] * c["E"] * rows * n, "flops": 4 * live * n * rows}


# ---- from the definition, in 64 bits ------------------------------------------------------------

def _exact_kept(x: torch.Tensor) -> torch.Tensor:
    v = x.double().unflatten(1, (-1, 32))
    big = v.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(torch.where(big > 0, big, 2.0 ** -130)))
    e = torch.where(torch.exp2(e) > big, e - 1, e)          # where the logarithm was rounded up to a whole number, or down
    e = torch.where(torch.exp2(e + 1) <= big, e + 1, e)
    unit = torch.exp2(torch.clamp(e, min=-127) - 6)
    low = torch.floor(v / unit)
    rest = v / unit - low
    up = (rest > 0.5) | ((rest == 0.5) & (low % 2 != 0))
    return ((low + up).clamp(-127, 127) * unit).flatten(1)


def exact(case: dict, seed: int):
    s, c = prepare(case, seed), case
    if c["kind"] == "kept":
        ff = c["ff"]
        h = s["gu"].double()[:, :ff] * torch.sigmoid(s["gu"].double()[:, :ff]) * s["gu"].double()[:, ff:]
        kept, gh = _exact_kept(s["gu"]), s["gh"].double()
        g, u = kept[:, :ff], kept[:, ff:]
        sig = torch.sigmoid(g)
        ggu = torch.cat((gh * u * (sig + g * sig * torch.sigmoid(-g)), gh * g * sig), 1)
        return h, ggu, g * sig * u, _exact_kept(s["x"])
    if c["kind"] == "adapter":
        offsets, which = s["requests"]
        out = s["y"].double()
        for i, j in enumerate(which):
            if j >= 0:
                rows = slice(offsets[i], offsets[i + 1])
                out[rows] += torch.einsum("rk,tk->tr", s["b"][j].double(), torch.einsum("kn,tn->tk", s["a"][j].double(), s["x"][rows].double())) * s["scale"][j].double()
        return out
    begin = [int(v) for v in s["offsets"]]
    if c["kind"] == "product":
        y = torch.zeros(s["x"].shape[0], c["rows"], dtype=torch.float64, device="cuda")
        for e in range(c["E"]):
            if begin[e + 1] > begin[e]:
                rows = slice(begin[e], begin[e + 1])
                y[rows] = torch.einsum("tn,rn->tr", s["x"][rows].double(), s["w"][e].double())
        return y
    gx = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    gw = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        rows = slice(begin[e], begin[e + 1])
        gy = s["gy"][rows].double()
        gx[rows] = torch.einsum("tr,rn->tn", gy, s["w"][e].double())
        gw[e] = torch.einsum("tr,tn->rn", gy, s["x"][rows].double())
    return gx, gw
