"""Benchmark cases of the scoring operators: the matrix product in 8-bit
integers with a scale per token and per channel (``i8_linear``,
``i8_quantize`` + ``i8_matmul``), log probabilities of given tokens with
entropy and top alternatives (``token_logprobs``), and the two joined at the
language-model head (``i8_head_logprobs``).

``run`` computes a case in plain torch operations, or with ``own`` set through
har_cuda.  Definitions:

* quantised row: s = max|x| / 127 and q = round(x / s), both quotients rounded
  to f32 and halves to even; a row of zeros has s = 0 and q = 0;
* product: y[m][n] = f32(sum_k q_x[m][k] q_w[n][k]) * f32(s_x[m] * s_w[n]), the
  sum exact, then rounded to y's type;
* distribution of a row of logits x: with M = max x and Z = sum exp(x - M),
  log p_i = (x_i - M) - log Z and H = log Z - sum exp(x - M) (x - M) / Z; a
  logit of -inf is a masked token (probability 0), a row of them alone has
  log p = -inf and H = 0; top alternatives by value, then lower index; a given
  token of -1 is padding and scores 0.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token through a projection of a 2048-wide model: launch latency counts
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 2048, "pad": 0, "x": "f32", "y": "f32"},
        # one token through a head of 131072 rows: the weights' bytes are all there is
        {"name": "linear_head", "op": "linear", "m": 1, "n": 131072, "k": 4096, "pad": 0, "x": "f32", "y": "f32"},
        # a decode batch through a head: weight bytes still, but 48 rows to multiply
        {"name": "linear_batch", "op": "linear", "m": 48, "n": 65536, "k": 2048, "pad": 0, "x": "bf16", "y": "f32"},
        # ragged sizes, rows that are slices of a wider buffer
        {"name": "linear_odd", "op": "linear", "m": 777, "n": 5003, "k": 1999, "pad": 7, "x": "f16", "y": "f16"},
        # a long prompt through a dense projection: arithmetic bound
        {"name": "linear_prompt", "op": "linear", "m": 8192, "n": 8192, "k": 4096, "pad": 0, "x": "bf16", "y": "bf16"},
        # a prompt quantised once for two projections (gate and up)
        {"name": "linear_pair", "op": "pair", "m": 512, "n": 2048, "k": 2048, "pad": 0, "x": "f32", "y": "bf16"},
        # one sequence's next-token distribution with 20 alternatives
        {"name": "logprobs_token", "op": "logprobs", "t": 1, "v": 131072, "x": "f32", "given": 1, "top": 20, "masked": 0.0},
        # every position of a prompt, 16-bit logits
        {"name": "logprobs_prompt", "op": "logprobs", "t": 4096, "v": 131072, "x": "bf16", "given": 1, "top": 5, "masked": 0.0},
        # odd vocabulary, constrained decoding: most tokens masked, one row empty, several answers per row
        {"name": "logprobs_odd", "op": "logprobs", "t": 301, "v": 50021, "x": "f16", "given": 4, "top": 20, "masked": 0.9},
        # a small batch scored from its hidden states
        {"name": "head_batch", "op": "head", "t": 8, "v": 65536, "k": 2048, "x": "f32", "given": 1, "top": 20},
        # odd vocabulary and row count, two answers per row
        {"name": "head_odd", "op": "head", "t": 203, "v": 50021, "k": 1999, "x": "f16", "given": 2, "top": 3},
        # a prompt scored from its hidden states: logits of 1 GB if they were kept
        {"name": "head_prompt", "op": "head", "t": 2048, "v": 131072, "k": 2048, "x": "bf16", "given": 1, "top": 5},
    ]


def _spread(rng, lo, hi, grain=1):
    """A size of [lo, hi], even over its logarithm; about half of them odd sizes."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if grain > 1 and rng.random() < 0.5:
        n = max(grain, n // grain * grain)
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["linear", "linear", "pair", "logprobs", "logprobs", "head", "head"])
    x = rng.choice(["f32", "f16", "bf16"])
    if op in ("linear", "pair"):
        m, k = _spread(rng, 1, 8192), _spread(rng, 64, 8192, 128)
        most = min(131072 if op == "linear" else 16384, 8192 * 8192 * 4096 // (m * k), (1 << 28) // m)
        n = _spread(rng, 64, max(64, most), 128)
        return {"op": op, "m": m, "n": n, "k": k, "pad": rng.choice([0, 0, 3, 8]), "x": x,
                "y": rng.choice(["f32", "f16", "bf16"])}
    given, top = rng.choice([0, 1, 1, 3]), rng.choice([0, 1, 5, 20, 32])
    if given + top == 0:
        given = 1
    if op == "logprobs":
        t = _spread(rng, 1, 4096)
        v = _spread(rng, 300, min(262144, (1 << 29) // t), 64)
        return {"op": op, "t": t, "v": v, "x": x, "given": given, "top": top,
                "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
    t, k = _spread(rng, 1, 2048), _spread(rng, 256, 4096, 128)
    v = _spread(rng, 1000, min(131072, 2048 * 131072 * 2048 // (t * k)), 64)
    return {"op": op, "t": t, "v": v, "k": k, "x": x, "given": given, "top": top}


# ---- inputs -------------------------------------------------------------------------


def _rows(gen, m, k, pad, dtype):
    """Token rows as a model's layers have them: normal, a few channels 8 times
    larger.  With padding they are slices of wider rows."""
    x = torch.randn(m, k + pad, device="cuda", generator=gen)
    x[:, :: max(1, k // 5)] *= 8
    return x.to(dtype)[:, :k]


def _weights(gen, n, k, spread):
    """Normal weights in 8 bits with a scale per channel: rows start at
    multiples of 16 bytes, as a program that lays them out once keeps them."""
    w = torch.randn(n, k, device="cuda", generator=gen)
    scale = w.abs().amax(1) * torch.rand(n, device="cuda", generator=gen).add_(0.5)
    q = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    q[:, :k] = torch.round(w.mul_((127 / scale)[:, None])).clamp_(-127, 127)
    return q[:, :k], scale.mul_(spread / 127)


def _given(gen, t, v, n):
    """Given tokens; the last row of several is padding."""
    tok = torch.randint(0, v, (t, n), device="cuda", generator=gen, dtype=torch.int32)
    if t > 1:
        tok[t - 1] = -1
    return tok


def _out(t, given, top):
    f = dict(dtype=torch.float32, device="cuda")
    return {"logprobs": torch.empty(t, given, **f), "entropy": torch.empty(t, **f),
            "top_ids": torch.empty(t, top, dtype=torch.int32, device="cuda"),
            "top_logprobs": torch.empty(t, top, **f)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op in ("linear", "pair"):
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _rows(gen, m, k, case["pad"], DTYPES[case["x"]])
        s["w"] = [_weights(gen, n, k, 0.02) for _ in range(2 if op == "pair" else 1)]
        s["y"] = [torch.empty(m, n, dtype=DTYPES[case["y"]], device="cuda") for _ in s["w"]]
        if op == "pair":
            s["q"] = torch.empty(m, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
            s["scale"] = torch.empty(m, dtype=torch.float32, device="cuda")
    elif op == "logprobs":
        t, v = case["t"], case["v"]
        x = torch.randn(t, v, device="cuda", generator=gen).mul_(2.5)
        x.scatter_add_(1, torch.randint(0, v, (t, 8), device="cuda", generator=gen),
                       torch.rand(t, 8, device="cuda", generator=gen).mul_(12))
        if case["masked"]:
            x.masked_fill_(torch.rand(t, v, device="cuda", generator=gen) < case["masked"], -math.inf)
            if t > 2:
                x[t // 2] = -math.inf
        s["x"] = x.to(DTYPES[case["x"]])
        s["tokens"] = _given(gen, t, v, case["given"])
        s["out"] = _out(t, case["given"], case["top"])
    else:
        t, v, k = case["t"], case["v"], case["k"]
        s["x"] = _rows(gen, t, k, 0, DTYPES[case["x"]])
        s["w"] = [_weights(gen, v, k, 2.5 / math.sqrt(k))]
        s["tokens"] = _given(gen, t, v, case["given"])
        s["out"] = _out(t, case["given"], case["top"])
    if own:
        s["ctx"] = _context()
        if "w" in s:
            s["handles"] = [s["ctx"].wrap_i8(q, scale) for q, scale in s["w"]]
    return s


_ctx = None


def _context():
    """The program's one context, on the stream that torch works on."""
    global _ctx
    if _ctx is None:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "remora-lab_b200"))
        import har_cuda
        _ctx = har_cuda.Context(0)
    return _ctx


# ---- the plain forms ------------------------------------------------------------------


def _quantize(x):
    x = x.float()
    scale = x.abs().amax(1) / torch.full((), 127.0, device=x.device)
    q = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0)
    return torch.round(q).clamp_(-127, 127), scale


def _slices(q):
    """[rows][k] -> [k / 1024][rows][1024], zeros behind the last: a slice's
    integer products stay below 2^24, so its f32 sums are exact."""
    rows, k = q.shape
    out = torch.zeros(rows, (k + 1023) // 1024 * 1024, device=q.device)
    out[:, :k] = q
    return out.view(rows, -1, 1024).transpose(0, 1)


def _product(q, scale, wq, wscale):
    parts = torch.bmm(_slices(q), _slices(wq).transpose(1, 2))
    acc = parts[0] if parts.shape[0] == 1 else parts.sum(0, dtype=torch.float64).float()
    return acc * (scale[:, None] * wscale[None, :])


def _distribution(x, tokens, top):
    x = x.float()
    v = x.shape[1]
    biggest = x.amax(1, keepdim=True)
    empty = biggest == -math.inf
    d = x - torch.where(empty, 0.0, biggest)
    e = torch.exp(d)
    z = torch.where(empty, 1.0, e.sum(1, keepdim=True, dtype=torch.float64))
    logz = torch.log(z)
    entropy = torch.where(empty, 0.0, logz - (e * torch.where(e > 0, d, 0.0)).sum(1, keepdim=True, dtype=torch.float64) / z)
    given = torch.gather(d, 1, tokens.clamp(min=0).long()) - logz
    given = torch.where(tokens < 0, 0.0, given)
    # keys in the order of (value, lower index): unique, so the largest are one answer
    bits = (x + 0.0).view(torch.int32).long()
    keys = torch.where(bits < 0, -2147483649 - bits, bits) * 262144 + (262143 - torch.arange(v, device=x.device))
    ids = 262143 - torch.topk(keys, min(top, v), dim=1).values % 262144
    best = torch.gather(d, 1, ids) - logz
    return {"logprobs": given.float(), "entropy": entropy[:, 0].float(), "top_ids": ids.int(), "top_logprobs": best.float()}


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        ctx = state["ctx"]
        if op == "linear":
            return ctx.i8_linear(state["handles"][0], state["x"], state["y"][0])
        if op == "pair":
            ctx.i8_quantize(state["x"], state["q"], state["scale"])
            return [ctx.i8_matmul(w, state["q"], state["scale"], y) for w, y in zip(state["handles"], state["y"])]
        o = state["out"]
        out = (o["logprobs"], o["entropy"], o["top_ids"], o["top_logprobs"])
        if op == "logprobs":
            ctx.token_logprobs(state["x"], state["tokens"], *out)
        else:
            ctx.i8_head_logprobs(state["handles"][0], state["x"], state["tokens"], *out)
        return o
    if op == "logprobs":
        return _distribution(state["x"], state["tokens"], case["top"])
    q, scale = _quantize(state["x"])
    if op == "head":
        return _distribution(_product(q, scale, *state["w"][0]), state["tokens"], case["top"])
    y = [_product(q, scale, *w).to(DTYPES[case["y"]]) for w in state["w"]]
    return y[0] if op == "linear" else y


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    op = case["op"]
    if op in ("linear", "pair"):
        m, n, k, w = case["m"], case["n"], case["k"], 2 if op == "pair" else 1
        return {"bytes": m * k * SIZE[case["x"]] + w * (n * k + 4 * n + m * n * SIZE[case["y"]]),
                "flops": 2 * w * m * n * k}
    t, v = case["t"], case["v"]
    small = t * (8 * case["given"] + 4 + 8 * case["top"])
    if op == "logprobs":
        # a subtraction, an exponential, two sums and a comparison for each logit
        return {"bytes": t * v * SIZE[case["x"]] + small, "flops": 5 * t * v}
    k = case["k"]
    return {"bytes": t * k * SIZE[case["x"]] + v * k + 4 * v + small, "flops": 2 * t * v * k + 5 * t * v}


# ---- the definitions in 64 bits -----------------------------------------------------------


def _product64(x, wq, wscale):
    x = x.double()
    scale = (x.abs().max(dim=1).values / 127).float().double()
    levels = (x / scale.unsqueeze(1)).float().nan_to_num(0.0, 0.0, 0.0).double()
    levels = levels.round().clamp(-127, 127)
    return (levels @ wq.double().t()).mul_(scale.unsqueeze(1)).mul_(wscale.double())


def _distribution64(x, tokens, top):
    """From torch.logsumexp's definition, log p = x - log sum exp x, in 64 bits."""
    lse = torch.logsumexp(x, 1, keepdim=True)
    none = torch.isneginf(lse)
    logp = torch.where(none, -math.inf, x - torch.where(none, 0.0, lse))
    best = logp.topk(top, 1).values
    given = logp.gather(1, tokens.long().clamp(min=0)).masked_fill(tokens < 0, 0.0)
    p = logp.exp()
    entropy = -(p * logp.masked_fill_(p == 0, 0.0)).sum(1)
    return {"logprobs": given, "entropy": entropy, "top_ids": None, "top_logprobs": best}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _distribution64(s["x"].double(), s["tokens"], case["top"])
    y = [_product64(s["x"], *w) for w in s["w"]]
    if case["op"] == "head":
        return _distribution64(y[0], s["tokens"], case["top"])
    return y[0] if case["op"] == "linear" else y
