"""Performance cases of the operators around an MoE block whose experts are not GGUF-quantised: what a program that
serves bf16, fp16 or 8-bit floating point experts asks of this package, as functions that a timing harness calls
(listed, draw, prepare, run, work, exact).

Five kinds of call:
  norm     ops.block_norm: the norm after a block, its gate, the scaled residual add and the norm before the next block
  gateup   ops.expert_gateup: gate and up products of the routed rows, grouped by expert, with SiLU(gate) * up
  proj     ops.expert_proj: the down product of the pairs' activation rows, grouped by expert
  rows     ops.fp8_rows: rows as e4m3 codes with one scale for each 128 values
  matmul   ops.fp8_matmul: rows times an e4m3 matrix with one scale for each block of 128 x 128

`own` chooses between the package's kernels and the plain form, which is elementary torch in 32 bits. Geometry "full" is
hidden 2048, ffn 768, 128 experts; "small" is hidden 1024, ffn 512, 32 experts; both route to 8 experts. The routing
tables are the package's: pair p = token * 8 + slot, pair_idx[E][stride] with the pairs of each expert in ascending
order and -1 behind them, pair_cnt[E].
"""
from __future__ import annotations

import math
import random

import torch

own = False

GEOMETRY = {"full": (128, 2048, 768), "small": (32, 1024, 512)}  # experts, hidden, ffn
TOP_K = 8
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "none": 0}
EPS = 1e-6
GROUP = 128           # values that share a scale
E4M3_MAX = 448.0
PER_MAX = 2.232142857142857e-3  # 1 / 448, rounded to f32 where it is used
SMALLEST = 2.0 ** -100  # groups whose largest value is below this are stored as zeros with a zero scale


def _norm(name, tokens, hidden, stream, block, gate, after, before):
    """stream, block: types of the residual stream and of the block's output ("none": only the norm before a block);
    gate: none, channel, row or full; after: the block's output is normalised first; before: type of the normalised
    rows for the next block ("none": there is no next block)."""
    return {"name": name, "kind": "norm", "tokens": tokens, "hidden": hidden, "stream": stream, "block": block, "gate": gate,
            "after": after, "before": before}


def _expert(name, kind, tokens, weights, out, routing, geometry="full"):
    return {"name": name, "kind": kind, "tokens": tokens, "weights": weights, "out": out, "routing": routing, "geometry": geometry}


def _matmul(name, m, n_out, n_in, dtype, out):
    return {"name": name, "kind": "matmul", "m": m, "n_out": n_out, "n_in": n_in, "dtype": dtype, "out": out}


def listed():
    return [
        # one decode step's hand-over from a block to the next: launch latency
        _norm("norm_t1", 1, 2048, "bf16", "f32", "none", True, "bf16"),
        # a short prompt through a block with a gate per token and an odd width, f32 residual stream
        _norm("norm_t301_gated", 301, 1000, "f32", "bf16", "row", True, "f16"),
        # many prompts at once, a gate per channel, the next block reads 8-bit rows
        _norm("norm_t16384_fp8", 16384, 2048, "bf16", "bf16", "channel", True, "e4m3"),
        # a single user's token: eight experts' gate and up matrices are read
        _expert("gateup_b1", "gateup", 1, "bf16", "bf16", "uniform"),
        # a small batch through the down matrices of a smaller model
        _expert("proj_b37_small", "proj", 37, "f16", "f32", "zipf", "small"),
        # the usual prefill chunk with popular and rare experts
        _expert("gateup_t512_zipf", "gateup", 512, "bf16", "bf16", "zipf"),
        # the same chunk over 8-bit experts
        _expert("gateup_t512_fp8", "gateup", 512, "e4m3", "bf16", "zipf"),
        # a long ragged prompt through the down matrices
        _expert("proj_t4001", "proj", 4001, "bf16", "f32", "zipf"),
        # many prompts at once: the largest grouped product
        _expert("gateup_t16384", "gateup", 16384, "bf16", "bf16", "uniform"),
        # one row times one 8-bit matrix, the smallest unit of a dense layer
        _matmul("matmul_m1", 1, 2048, 2048, "bf16", "f32"),
        # a short prompt through a dense layer, odd numbers of rows and columns
        _matmul("matmul_m301", 301, 1000, 2048, "bf16", "bf16"),
        # many prompts at once through a dense layer
        _matmul("matmul_m8192", 8192, 4096, 4096, "bf16", "bf16"),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["norm", "norm", "gateup", "gateup", "proj", "proj", "rows", "matmul", "matmul", "matmul"])
    if kind == "norm":
        block = rng.choice(["none", "bf16", "f16", "f32"])
        before = "bf16" if block == "none" else rng.choice(["none", "bf16", "f16", "f32", "e4m3"])
        step = rng.choice([1, 8, 128])
        hidden = step * _log_int(rng, max(1, 64 // step), 16384 // step)
        case = _norm("", _log_int(rng, 1, min(16384, (1 << 25) // hidden)), hidden, rng.choice(["f32", "bf16", "bf16"]),
                     block, rng.choice(["none", "channel", "row", "full"]), rng.random() < 0.7, before)
    elif kind == "rows":
        case = {"name": "", "kind": "rows", "tokens": _log_int(rng, 1, 16384), "hidden": 8 * _log_int(rng, 16, 512),
                "dtype": rng.choice(["f32", "bf16", "f16"])}
    elif kind == "matmul":
        case = _matmul("", _log_int(rng, 1, 4096), _log_int(rng, 100, 4096), 16 * _log_int(rng, 8, 256), rng.choice(["f32", "bf16", "f16"]),
                       rng.choice(["bf16", "bf16", "f32", "f16"]))
    else:
        weights = rng.choice(["bf16", "f16", "e4m3", "e4m3"])
        routing = rng.choice(["uniform", "zipf"])
        case = _expert("", kind, _log_int(rng, 1, 4096 if routing == "zipf" else 12000), weights,
                       rng.choice(["bf16", "f16"] if kind == "gateup" else ["f32", "bf16"]), routing, rng.choice(["full", "full", "small"]))
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------------------- inputs

def _routing(E: int, tokens: int, routing: str, g):
    """Routing tables of `tokens` tokens with eight distinct experts each (a uniform or Zipf(1.1) popularity), and the
    largest number of pairs that one expert got."""
    score = torch.rand((tokens, E), device="cuda", generator=g).log_().neg_().log_().neg_()
    if routing == "zipf":
        p = torch.arange(1, E + 1, device="cuda").double().pow(-1.1)
        score += torch.log(p / p.sum()).float()[torch.randperm(E, device="cuda", generator=g)]
    pair_exp = score.topk(TOP_K, dim=1).indices.reshape(-1)
    cnt = torch.bincount(pair_exp, minlength=E)
    order = torch.argsort(pair_exp, stable=True)
    start = torch.cumsum(cnt, 0) - cnt
    slot = torch.arange(tokens * TOP_K, device="cuda") - start[pair_exp[order]]
    idx = torch.full((E, tokens), -1, dtype=torch.int32, device="cuda")
    idx[pair_exp[order], slot] = order.int()
    return {"pair_idx": idx, "pair_cnt": cnt.int(), "most": int(cnt.max())}


def _weight(shape, kind: str, g):
    """A matrix (or one for each expert) with a standard deviation of 0.02, and its scales where it is held in 8 bits."""
    w = torch.randn(shape, device="cuda", generator=g).mul_(0.02)
    if kind != "e4m3":
        return w.to(DTYPE[kind]), None
    n, k = shape[-2:]
    nb, kb = -(-n // GROUP), -(-k // GROUP)
    pad = torch.nn.functional.pad(w, (0, kb * GROUP - k, 0, nb * GROUP - n)).unflatten(-1, (kb, GROUP)).unflatten(-3, (nb, GROUP))
    scale = pad.abs().amax(dim=(-3, -1)) / E4M3_MAX
    codes = (pad / scale[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :n, :k]
    return codes.contiguous().to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def rows(n, k, dtype):
        return torch.randn((n, k), device="cuda", generator=g).to(DTYPE[dtype])

    kind = case["kind"]
    if kind == "norm":
        T, H = case["tokens"], case["hidden"]
        w = [(1.0 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2)]
        gate = {"none": None, "channel": (H,), "row": (T, 1), "full": (T, H)}[case["gate"]]
        block = case["block"] != "none"
        return {"case": case, "x": rows(T, H, case["stream"]), "y": 0.3 * rows(T, H, case["block"]) if block else None,
                "after": w[0] if block and case["after"] else None, "before": w[1] if case["before"] != "none" else None,
                "gate": torch.randn(gate, device="cuda", generator=g).to(torch.bfloat16) if block and gate else None, "scale": 0.7}
    if kind == "rows":
        return {"case": case, "x": rows(case["tokens"], case["hidden"], case["dtype"])}
    if kind == "matmul":
        w, scale = _weight((case["n_out"], case["n_in"]), "e4m3", g)
        return {"case": case, "x": rows(case["m"], case["n_in"], case["dtype"]), "w": w, "scale": scale}
    E, H, F = GEOMETRY[case["geometry"]]
    T = case["tokens"]
    state = {"case": case, **_routing(E, T, case["routing"], g)}
    held = "bf16" if case["weights"] == "e4m3" else case["weights"]   # the rows come in 16 bits
    if kind == "gateup":
        state["x"] = rows(T, H, held)
        state["wg"], state["sg"] = _weight((E, F, H), case["weights"], g)
        state["wu"], state["su"] = _weight((E, F, H), case["weights"], g)
    else:
        state["x"] = 0.3 * rows(T * TOP_K, F, held)
        state["wd"], state["sd"] = _weight((E, H, F), case["weights"], g)
    return state


# ---------------------------------------------------------------------------------------------------------- run

def _plain_codes(x):
    """Rows in groups of 128 values (zeros behind the last): e4m3 codes and one f32 scale for each group."""
    k = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -k % GROUP)).unflatten(-1, (-1, GROUP))
    most = v.abs().amax(-1)
    scale = torch.where(most < SMALLEST, 0.0, most * PER_MAX)
    inverse = torch.where(most < SMALLEST, 0.0, 1.0 / scale)
    return (v * inverse[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).flatten(-2)[..., :k], scale


def _plain_values(codes, scale):
    return codes.float() * scale.repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]


def _plain_weight(w, scale):
    if scale is None:
        return w.float()
    return w.float() * scale.repeat_interleave(GROUP, -1)[..., :w.shape[-1]].repeat_interleave(GROUP, -2)[..., :w.shape[-2], :]


def _plain_rms(v, w):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w.float()


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    stream = None
    if s["y"] is not None:
        y = s["y"].float()
        if s["after"] is not None:
            y = _plain_rms(y, s["after"])
        if s["gate"] is not None:
            y = y * (1.0 / (1.0 + torch.exp(-s["gate"].float())))
        x = x + s["scale"] * y
        stream = x.to(s["x"].dtype)
    if s["before"] is None:
        return stream, None
    h = _plain_rms(x, s["before"])
    return stream, _plain_codes(h) if case["before"] == "e4m3" else h.to(DTYPE[case["before"]])


def _plain_rows(s):
    """The rows as the product sees them, in f32."""
    return _plain_values(*_plain_codes(s["x"])) if s["case"]["weights"] == "e4m3" else s["x"].float()


def _plain_scatter(s, y):
    """[E][most][N] -> [pairs][N] in the output's type; what lies behind an expert's last pair is dropped."""
    n_pairs = s["case"]["tokens"] * TOP_K
    idx = s["pair_idx"][:, :s["most"]].long()
    out = torch.zeros((n_pairs + 1, y.shape[-1]), dtype=DTYPE[s["case"]["out"]], device="cuda")
    out[torch.where(idx >= 0, idx, n_pairs)] = y.to(out.dtype)
    return out[:n_pairs]


def _plain_gateup(s):
    tok = s["pair_idx"][:, :s["most"]].long().clamp_(min=0) // TOP_K
    x = _plain_rows(s)[tok]
    gate = torch.bmm(x, _plain_weight(s["wg"], s["sg"]).transpose(1, 2))
    up = torch.bmm(x, _plain_weight(s["wu"], s["su"]).transpose(1, 2))
    return _plain_scatter(s, gate / (1.0 + torch.exp(-gate)) * up)


def _plain_proj(s):
    x = _plain_rows(s)[s["pair_idx"][:, :s["most"]].long().clamp_(min=0)]
    return _plain_scatter(s, torch.bmm(x, _plain_weight(s["wd"], s["sd"]).transpose(1, 2)))


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from kanjoos_b200 import ops
        if kind == "norm":
            return ops.block_norm(state["x"], state["y"], post_w=state["after"], gate=state["gate"], gate_sigmoid=True, alpha=state["scale"],
                                  pre_w=state["before"], eps=EPS,
                                  norm_dtype=torch.float8_e4m3fn if case["before"] == "e4m3" else DTYPE.get(case["before"], torch.bfloat16))
        if kind == "rows":
            return ops.fp8_rows(state["x"])
        if kind == "matmul":
            return ops.fp8_matmul(state["w"], state["scale"], state["x"], out_dtype=DTYPE[case["out"]])
        if kind == "gateup":
            return ops.expert_gateup(state["x"], state["wg"], state["wu"], state["pair_idx"], state["pair_cnt"], case["tokens"] * TOP_K, TOP_K,
                                     gate_scale=state["sg"], up_scale=state["su"], out_dtype=DTYPE[case["out"]])
        return ops.expert_proj(state["x"], state["wd"], state["pair_idx"], state["pair_cnt"], case["tokens"] * TOP_K, scale=state["sd"],
                               out_dtype=DTYPE[case["out"]])
    if kind == "norm":
        return _plain_norm(state)
    if kind == "rows":
        return _plain_codes(state["x"])
    if kind == "matmul":
        x = _plain_values(*_plain_codes(state["x"]))
        return (x @ _plain_weight(state["w"], state["scale"]).t()).to(DTYPE[case["out"]])
    return _plain_gateup(state) if kind == "gateup" else _plain_proj(state)


# ------------------------------------------------------------------------------------------- what a pass needs

def _distinct(E: int, tokens: int, routing: str) -> float:
    """Expected number of experts that at least one of the tokens routes to."""
    z = [i ** -1.1 for i in range(1, E + 1)]
    p = [TOP_K / E] * E if routing == "uniform" else [min(0.98, TOP_K * v / sum(z)) for v in z]
    return sum(1.0 - (1.0 - v) ** tokens for v in p)


def work(case):
    kind = case["kind"]
    if kind == "norm":
        T, H = case["tokens"], case["hidden"]
        block = case["block"] != "none"
        per = SIZE[case["stream"]] * (2 if block else 1) + SIZE[case["block"]] + SIZE[case["before"]]
        extra = {"none": 0, "channel": H, "row": T, "full": T * H}[case["gate"]] * 2 if block else 0
        return {"bytes": T * H * per + extra + 4 * H, "flops": T * H * 12}
    if kind == "rows":
        return {"bytes": case["tokens"] * case["hidden"] * (SIZE[case["dtype"]] + 1 + 4 / GROUP), "flops": case["tokens"] * case["hidden"] * 3}
    if kind == "matmul":
        m, n, k = case["m"], case["n_out"], case["n_in"]
        return {"bytes": n * k + m * k * SIZE[case["dtype"]] + m * n * SIZE[case["out"]], "flops": 2.0 * m * n * k}
    E, H, F = GEOMETRY[case["geometry"]]
    T, w = case["tokens"], case["weights"]
    P = T * TOP_K
    mats, rows, k, n = (2, T, H, F) if kind == "gateup" else (1, P, F, H)
    return {"bytes": _distinct(E, T, case["routing"]) * mats * H * F * SIZE[w] + rows * k * 2 + P * n * SIZE[case["out"]],
            "flops": 2.0 * P * mats * H * F}


# ------------------------------------------------------------------------------- the definition, in 64 bits

def _exact_quantised(x):
    """(codes as values, scales) of rows, from the definition: the scale is the f32 product of the largest magnitude and
    the f32 nearest to 1 / 448, a code the e4m3 value nearest to the f32 product of the value and the f32 inverse of the
    scale, ties to the even one. Codes are discrete, so these roundings are part of the definition: 16-bit values over
    16-bit maxima often end on a tie."""
    x = x.double()
    T, K = x.shape
    codes, scales = torch.zeros_like(x), []
    for b in range(0, K, GROUP):
        part = x[:, b:b + GROUP]
        most = part.abs().max(dim=1, keepdim=True).values
        scale = (most * torch.tensor(PER_MAX, dtype=torch.float32).double()).float().double()
        v = torch.where(most >= SMALLEST, (part * (1.0 / scale).float().double()).float().double(), torch.zeros_like(part))
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        codes[:, b:b + GROUP] = (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
        scales.append(torch.where(most >= SMALLEST, scale, torch.zeros_like(scale)))
    return codes, torch.cat(scales, dim=1)


def _exact_held(x):
    codes, scale = _exact_quantised(x)
    for b in range(scale.shape[1]):
        codes[:, b * GROUP:(b + 1) * GROUP] *= scale[:, b:b + 1]
    return codes


def _exact_matrix(w, scale):
    w = w.double()
    if scale is not None:
        for i in range(scale.shape[0]):
            for j in range(scale.shape[1]):
                w[i * GROUP:(i + 1) * GROUP, j * GROUP:(j + 1) * GROUP] *= scale[i, j].double()
    return w


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x, stream = s["x"].double(), None
        if s["y"] is not None:
            y = s["y"].double()
            if s["after"] is not None:
                y = y / torch.sqrt((y * y).sum(dim=1, keepdim=True) / y.shape[1] + EPS) * s["after"].double()
            if s["gate"] is not None:
                y = y * torch.sigmoid(s["gate"].double())
            x = stream = x + s["scale"] * y   # the next norm reads the stream before it is rounded to its type
        if s["before"] is None:
            return stream, None
        h = x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / x.shape[1] + EPS) * s["before"].double()
        return stream, _exact_quantised(h) if case["before"] == "e4m3" else h
    if kind == "rows":
        return _exact_quantised(s["x"])
    if kind == "matmul":
        return _exact_held(s["x"]) @ _exact_matrix(s["w"], s["scale"]).t()
    x = _exact_held(s["x"]) if case["weights"] == "e4m3" else s["x"].double()
    P = case["tokens"] * TOP_K
    E, H, F = GEOMETRY[case["geometry"]]
    out = torch.zeros((P, F if kind == "gateup" else H), dtype=torch.float64, device="cuda")
    for e, n in enumerate(s["pair_cnt"].tolist()):
        if n == 0:
            continue
        pairs = s["pair_idx"][e, :n].long()
        if kind == "gateup":
            rows = x[pairs // TOP_K]
            gate = rows @ _exact_matrix(s["wg"][e], None if s["sg"] is None else s["sg"][e]).t()
            up = rows @ _exact_matrix(s["wu"][e], None if s["su"] is None else s["su"][e]).t()
            out[pairs] = gate * torch.sigmoid(gate) * up
        else:
            out[pairs] = x[pairs] @ _exact_matrix(s["wd"][e], None if s["sd"] is None else s["sd"][e]).t()
    return out
