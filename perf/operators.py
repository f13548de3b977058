"""The predictive operators as they are measured: inputs, plain forms, and the calls that a user makes.

Three operators answer with what the samplers have drawn (mcmc_amd/predictive.py):

  quantize   rows of a matrix in 8 bits (e4m3), with a power of two for each block of 128 columns of a row
  product    X . Theta^T of rows with posterior draws held that way: the predictor of every row under every draw
  draw       one column for each row of log weights, from a given random number: temperature, top-k, top-p, min-p

A case is a dict of plain values; `own` chooses between the plain forms here and the package's calls.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the double design matrix as the samplers keep it, column by column, made ready once for prediction
        {"name": "quantize design matrix", "op": "quantize", "rows": 1_000_003, "cols": 64, "type": "f64", "order": "columns"},
        # a wide matrix that is already in 16 bits
        {"name": "quantize wide rows", "op": "quantize", "rows": 8192, "cols": 4096, "type": "bf16", "order": "rows"},
        # one new observation under the draws that 64 chains kept: the call whose latency a user waits for
        {"name": "product one row", "op": "product", "rows": 1, "draws": 50_000, "cols": 128, "type": "f32", "out": "f32", "ready": False},
        # one wide observation against many wide draws: the draws' bytes are all there is to it
        {"name": "product one wide row", "op": "product", "rows": 1, "draws": 8192, "cols": 8192, "type": "bf16", "out": "f32", "ready": False},
        # a held-out set of the benchmark's width under a thinned chain: the output's bytes bound it
        {"name": "product held-out set", "op": "product", "rows": 200_000, "draws": 1000, "cols": 64, "type": "f32", "out": "bf16", "ready": False},
        # wide rows, quantized within the call, and predictors that are summed on: all the accuracy of 32 bits
        {"name": "product wide rows", "op": "product", "rows": 4096, "draws": 4096, "cols": 4096, "type": "bf16", "out": "f32", "ready": False},
        # the largest: both sides are ready, the matrix cores' rate bounds it
        {"name": "product largest", "op": "product", "rows": 8192, "draws": 8192, "cols": 8192, "type": "bf16", "out": "bf16", "ready": True},
        # one observation, the draws of a short chain
        {"name": "draw one short row", "op": "draw", "rows": 1, "n": 1000, "type": "f32", "spread": 2.0, "masked": 0.0, "temperature": 0.8, "top_k": 40, "top_p": 0.9, "min_p": 0.0, "each": False},
        # one long row in 16 bits, where many weights are equal
        {"name": "draw one long row", "op": "draw", "rows": 1, "n": 131_072, "type": "bf16", "spread": 3.0, "masked": 0.0, "temperature": 0.7, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "each": False},
        # a batch with an odd length, without a top-k: the nucleus is looked for in the whole row
        {"name": "draw nucleus", "op": "draw", "rows": 64, "n": 50_001, "type": "f32", "spread": 2.5, "masked": 0.0, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "each": False},
        # many long rows, temperature alone: plain resampling by weight, bound by the reading of the weights
        {"name": "draw plain resampling", "op": "draw", "rows": 256, "n": 131_072, "type": "f32", "spread": 1.5, "masked": 0.0, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "each": False},
        # many short rows, a part of each masked, each with choices of its own
        {"name": "draw masked rows", "op": "draw", "rows": 4096, "n": 2000, "type": "f16", "spread": 3.0, "masked": 0.3, "temperature": 0.9, "top_k": 200, "top_p": 0.95, "min_p": 0.02, "each": True},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "draw", "draw"])
    if op == "quantize":
        cols = _log_uniform(rng, 3, 8192)
        rows = _log_uniform(rng, 1, min(1_000_000, 64_000_000 // cols))
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["f64", "f32", "bf16", "f16"]), "order": rng.choice(["rows", "rows", "columns"])}
    if op == "product":
        cols = _log_uniform(rng, 3, 8192)
        draws = _log_uniform(rng, 1, min(50_000, 64_000_000 // cols))
        rows = _log_uniform(rng, 1, max(1, min(200_000, 64_000_000 // cols, 200_000_000 // draws, 2 ** 37 // (cols * draws))))
        return {"op": op, "rows": rows, "draws": draws, "cols": cols, "type": rng.choice(["f32", "bf16", "f16"]), "out": rng.choice(["f32", "bf16", "f16"]), "ready": rng.random() < 0.3}
    n = _log_uniform(rng, 2, 262_144)
    return {"op": op, "rows": _log_uniform(rng, 1, min(4096, 2 ** 25 // n)), "n": n, "type": rng.choice(["f32", "bf16", "f16"]), "spread": rng.choice([0.5, 1.5, 3.0, 6.0]),
            "masked": rng.choice([0.0, 0.0, 0.3]), "temperature": rng.choice([0.5, 0.8, 1.0, 1.3]), "top_k": rng.choice([0, 1, 40, 1000]), "top_p": rng.choice([1.0, 0.95, 0.5]),
            "min_p": rng.choice([0.0, 0.0, 0.05]), "each": rng.random() < 0.4}


# ---------------------------------------------------------------- inputs

def _features(g, rows, cols, dtype):
    """Observations: a constant column, the others uniform, as in the framework's synthetic data."""
    x = torch.rand(rows, cols, generator=g, device="cuda", dtype=torch.float64 if dtype == torch.float64 else torch.float32)
    x[:, 0] = 1.0
    return x.to(dtype)


def _posterior(g, draws, cols):
    """Draws of a coefficient vector: a common centre, and a spread about it that differs from column to column."""
    centre = 0.5 * torch.randn(cols, generator=g, device="cuda")
    width = 0.02 + 0.2 * torch.rand(cols, generator=g, device="cuda")
    return centre + width * torch.randn(draws, cols, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "quantize":
        x = _features(g, case["rows"], case["cols"], TYPES[case["type"]])
        state["x"] = x.t().contiguous().t() if case["order"] == "columns" else x
    elif case["op"] == "product":
        # the draws are laid out once, when the chain has ended
        state["w"] = quantize_plain(_posterior(g, case["draws"], case["cols"]))
        x = _features(g, case["rows"], case["cols"], TYPES[case["type"]])
        state["x"] = quantize_plain(x) if case["ready"] else x
    else:
        rows, n = case["rows"], case["n"]
        z = case["spread"] * torch.randn(rows, n, generator=g, device="cuda")
        if case["masked"]:
            z = z.masked_fill(torch.rand(rows, n, generator=g, device="cuda") < case["masked"], -math.inf)
        state["z"] = z.to(TYPES[case["type"]])
        state["u"] = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        keys = ("temperature", "top_k", "top_p", "min_p")
        if case["each"]:  # every row has choices of its own around the case's
            r = torch.rand(4, rows, generator=g, device="cuda")
            state["temperature"] = case["temperature"] * (0.75 + 0.5 * r[0])
            state["top_k"] = (case["top_k"] * (0.5 + r[1])).to(torch.int32)
            state["top_p"] = 1.0 - (1.0 - case["top_p"]) * (0.5 + r[2])
            state["min_p"] = case["min_p"] * (0.5 + r[3])
        else:
            state.update({k: case[k] for k in keys})
    return state


# ---------------------------------------------------------------- plain forms

def quantize_plain(x):
    """(data, scale): e4m3 values of x / 2^k, columns padded with zeros to blocks of 128, and k + 127 for each block of
    a row, padded to whole groups of four. k is the least power from -96 to 119 that brings the block's largest magnitude
    to 448 or less; what is larger still, or not finite, becomes NaN."""
    x = x if x.dtype == torch.float64 else x.float()  # a double is rounded once, to 8 bits
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    top = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
    k = torch.where(top == 0, 0, torch.where(m <= 0.875, e - 9, e - 8).clamp(-96, 119))
    y = x * _power(-k, x.dtype)
    e = torch.frexp(y)[1].clamp(min=-5)  # the last place of e4m3: 2^-9 below 2^-6, three bits below the first above
    step = _power(e - 4, x.dtype)
    q = torch.round(y / step) * step
    q = torch.where(y.abs() <= 448, q, math.nan)
    scale = torch.full((rows, 4 * -(-blocks // 4)), 127, dtype=torch.uint8, device=x.device)
    scale[:, :blocks] = (k.squeeze(-1) + 127).to(torch.uint8)
    return q.view(rows, -1).to(torch.float8_e4m3fn), scale


def _power(k, dtype):
    """2^k, exactly, for whole k within the type's normal range."""
    return ((k.long() + 1023) << 52).view(torch.float64).to(dtype)


def dequantize_plain(q):
    data, scale = q
    blocks = data.shape[1] // BLOCK
    p = _power(scale[:, :blocks].long() - 127, torch.float32)
    return (data.float().view(data.shape[0], blocks, BLOCK) * p[:, :, None]).view(data.shape)


def product_plain(x, w, out):
    x = dequantize_plain(x if isinstance(x, tuple) else quantize_plain(x))
    return torch.matmul(x, dequantize_plain(w).t()).to(out)


def _each(v, z):
    return v.to(z.dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((z.shape[0], 1), float(v), dtype=z.dtype, device=z.device)


def draw_plain(z, u, temperature, top_k, top_p, min_p):
    """(column, its log probability) of each row. In 64 bits: a sum decides on which side of a border u falls."""
    z, u = z.double(), u.double()[:, None]
    n = z.shape[1]
    temperature, top_k, top_p, min_p = (_each(v, z) for v in (temperature, top_k, top_p, min_p))
    top = z.amax(-1, keepdim=True)
    w = torch.where(z == top, 1.0, torch.exp((z - top) / temperature))  # an empty weight stays empty at any temperature
    w = torch.where(z == -math.inf, 0.0, w)
    order = torch.sort(z, dim=-1, descending=True, stable=True)[1]  # equal weights: the lower column first
    ws = torch.gather(w, 1, order)
    place = torch.arange(n, device=z.device)[None, :]
    keep = (place < top_k) | (top_k <= 0)
    ws = torch.where(keep, ws, 0.0)
    reached = torch.cumsum(ws, -1)
    before = torch.nn.functional.pad(reached, (1, 0))[:, :-1]
    keep &= (top_p >= 1) | (before < top_p * reached[:, -1:]) | (place == 0)
    keep &= (ws >= min_p.clamp(max=1.0)) | (min_p <= 0)
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0.0)  # back in the columns' order
    reached = torch.cumsum(w, -1)
    total = reached[:, -1:]
    some = torch.where(w > 0, place, -1)
    column = torch.minimum((reached <= u * total).sum(-1, keepdim=True), some.amax(-1, keepdim=True))  # -1: nothing to draw
    logp = torch.log(torch.gather(w, 1, column.clamp(min=0)) / total)
    return column[:, 0], torch.where(column < 0, math.nan, logp)[:, 0].float()


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if own:
        from mcmc_amd import predictive

        if case["op"] == "quantize":
            q = predictive.quantize(state["x"])
            return q.data, q.scale
        if case["op"] == "product":
            x = predictive.Block8(*state["x"], case["cols"]) if case["ready"] else state["x"]
            return predictive.product(x, predictive.Block8(*state["w"], case["cols"]), TYPES[case["out"]])
        return predictive.draw(state["z"], state["u"], state["temperature"], state["top_k"], state["top_p"], state["min_p"])
    if case["op"] == "quantize":
        return quantize_plain(state["x"])
    if case["op"] == "product":
        return product_plain(state["x"], state["w"], TYPES[case["out"]])
    return draw_plain(state["z"], state["u"], state["temperature"], state["top_k"], state["top_p"], state["min_p"])


def _bytes8(rows, cols):
    """What a quantized matrix has to hold: a byte a value, and a byte a block."""
    return rows * cols + rows * -(-cols // BLOCK)


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * SIZE[case["type"]] + _bytes8(case["rows"], case["cols"]), "flops": 3 * n}
    if case["op"] == "product":
        m, n, k = case["rows"], case["draws"], case["cols"]
        x = _bytes8(m, k) if case["ready"] else m * k * SIZE[case["type"]]
        return {"bytes": x + _bytes8(n, k) + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    n = case["rows"] * case["n"]
    return {"bytes": n * SIZE[case["type"]] + case["rows"] * 20, "flops": 4 * n}  # a difference, a quotient, an exponential, a sum


# ---------------------------------------------------------------- the definition, in 64 bits

def _exact_rows8(x):
    """The values that the quantized rows stand for divided by their scales, and the scales' powers: by search in the
    list of all e4m3 values."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    wide = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    wide[:, :cols] = x.double()
    wide = wide.reshape(rows, blocks, BLOCK)
    top = wide.abs().nan_to_num(0.0, 0.0, 0.0).max(-1).values
    k = torch.ceil(torch.log2(top / 448.0)).clamp(-200, 200)  # may be one off beside a power of two
    k = torch.where(top > 448.0 * torch.exp2(k), k + 1, k)
    k = torch.where(top <= 448.0 * torch.exp2(k - 1), k - 1, k)
    k = torch.where(top > 0, k.clamp(-96, 119), 0.0)
    y = wide / torch.exp2(k)[:, :, None]
    code = torch.arange(127, dtype=torch.float64, device=x.device)
    e, m = torch.floor(code / 8), code % 8
    value = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))
    half = (value[1:] + value[:-1]) / 2
    below = torch.bucketize(y.abs(), half, right=False)  # a tie goes down here
    tie = (below < 126) & (y.abs() == half[below.clamp(max=125)]) & (below % 2 == 1)
    q = torch.copysign(value[below + tie.long()], y)
    return q, k


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        q, k = _exact_rows8(state["x"])
        codes = torch.full(quantize_shape(case), 127, dtype=torch.int64, device=q.device)
        codes[:, : k.shape[1]] = k.long() + 127
        return q.reshape(q.shape[0], -1), codes
    if case["op"] == "product":
        def values(data, scale):
            blocks = data.shape[1] // BLOCK
            return data.double() * torch.exp2(scale[:, :blocks].double() - 127.0).repeat_interleave(BLOCK, dim=1)

        if case["ready"]:
            x = values(*state["x"])
        else:
            q, k = _exact_rows8(state["x"])
            x = (q * torch.exp2(k)[:, :, None]).reshape(q.shape[0], -1)
        return torch.mm(x, values(*state["w"]).t().contiguous())
    return _exact_draw(state)


def quantize_shape(case):
    return case["rows"], 4 * -(-case["cols"] // (4 * BLOCK))


def _exact_draw(state):
    z, u = state["z"].double().cpu().numpy(), state["u"].double().cpu().numpy()
    each = [v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(len(z), float(v)) for v in (state["temperature"], state["top_k"], state["top_p"], state["min_p"])]
    columns, logs = np.zeros(len(z), np.int64), np.zeros(len(z))
    for i, (t, k, p, m) in enumerate(zip(*each)):
        order = np.lexsort((np.arange(z.shape[1]), -z[i]))
        some = z[i][order] > -np.inf
        weight = np.zeros(len(order))
        weight[some] = np.exp((z[i][order][some] - z[i][order[0]]) / t)
        if k > 0:
            order, weight = order[: int(k)], weight[: int(k)]
        if p < 1:
            last = np.searchsorted(np.cumsum(weight), p * np.sum(weight), side="left")
            most = last + 1
        else:
            most = len(order)
        if m > 0:
            most = min(most, int(np.sum(weight >= min(m, 1.0))))
        order, weight = order[:most], weight[:most]
        back = np.argsort(order)
        order, weight = order[back], weight[back]
        order, weight = order[weight > 0], weight[weight > 0]
        if len(order) == 0:
            columns[i], logs[i] = -1, np.nan
            continue
        reached = np.cumsum(weight)
        at = min(int(np.searchsorted(reached, u[i] * reached[-1], side="right")), len(order) - 1)
        columns[i], logs[i] = order[at], np.log(weight[at] / reached[-1])
    return torch.from_numpy(columns), torch.from_numpy(logs)
