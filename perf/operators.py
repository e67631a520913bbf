"""The operators of the scoring head, case by case: what is measured, in plain torch and through the library.

A causal language model re-orders retrieved pages by how likely it finds the question after each of them.  Its last
hidden states are normed and held in 8 bits, multiplied with a vocabulary matrix held in 4 bits, and the logits turned
into log probabilities of the question's tokens:

    quantize     rows to microscaled 4- or 8-bit floating point and back (a matrix as it is loaded, queries as they come)
    dequantize   microscaled rows read back
    norm         residual addition + root-mean-square norm, quantised to 8 bits, and read back
    matmul       8-bit (or 4-bit) rows times the transpose of 4-bit rows
    logprobs     log probabilities of given tokens, entropy, top alternatives

Microscaled rows: blocks of 32 elements share a power-of-two scale (8 bits, bias 127, 255 = NaN); the elements are
e2m1 (two a byte, the earlier one in the low half) or e4m3; rows are padded with zeros to a multiple of 128 elements."""
import math

import torch

own = False

BLOCK, PAD = 32, 128
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
ELEMENT = {"mxfp4": (2, 6.0, 7.0, 2), "mxfp8": (8, 448.0, 464.0, 4)}  # exponent and value of the largest, where the scale steps up, significant bits


def listed():
    return [
        # the keyword vectors of the sample run (34 unique keywords, the default encoder's width), quantised before a search
        {"name": "quantize 34x4096 fp32 to 8 bits", "op": "quantize", "n": 34, "d": 4096, "dtype": "fp32", "format": "mxfp8"},
        # a page index of a million rows, quantised as it is loaded
        {"name": "quantize 1Mx1024 bf16 to 4 bits", "op": "quantize", "n": 1_000_000, "d": 1024, "dtype": "bf16", "format": "mxfp4"},
        # the textbook's 4032 pages read back for a check or a re-scoring in full precision
        {"name": "dequantize 4032x4096 4 bits to fp32", "op": "dequantize", "n": 4032, "d": 4096, "dtype": "fp32", "format": "mxfp4"},
        # a large index held in 8 bits read back in half precision, at a width that is no multiple of the padding
        {"name": "dequantize 1Mx1000 8 bits to bf16", "op": "dequantize", "n": 1_000_000, "d": 1000, "dtype": "bf16", "format": "mxfp8"},
        # one new token of one sequence
        {"name": "norm 1x4096 bf16", "op": "norm", "n": 1, "d": 4096, "dtype": "bf16", "format": "mxfp8", "residual": True},
        # one page at the builder's truncation length
        {"name": "norm 8192x4096 bf16", "op": "norm", "n": 8192, "d": 4096, "dtype": "bf16", "format": "mxfp8", "residual": True},
        # the logits of one new token: the whole vocabulary matrix is read for it
        {"name": "matmul 1x131072x4096 8x4", "op": "matmul", "m": 1, "n": 131072, "k": 4096, "a": "mxfp8", "out": "fp32"},
        # a batch of queries against an index, both in 4 bits, odd numbers of rows
        {"name": "matmul 511x100003x768 4x4", "op": "matmul", "m": 511, "n": 100_003, "k": 768, "a": "mxfp4", "out": "fp32"},
        # the question tokens of a re-ranking batch
        {"name": "matmul 2048x131072x4096 8x4", "op": "matmul", "m": 2048, "n": 131072, "k": 4096, "a": "mxfp8", "out": "bf16"},
        # one new token: its yes / no answers and twenty alternatives
        {"name": "logprobs 1x131072 fp32 top 20", "op": "logprobs", "n": 1, "v": 131072, "dtype": "fp32", "tokens": 2, "top": 20, "masked": 0.0},
        # the question of one page, a vocabulary of odd size, part of it forbidden
        {"name": "logprobs 63x50257 fp16 top 5", "op": "logprobs", "n": 63, "v": 50257, "dtype": "fp16", "tokens": 1, "top": 5, "masked": 0.4},
        # the question tokens of a re-ranking batch
        {"name": "logprobs 2048x131072 bf16 top 1", "op": "logprobs", "n": 2048, "v": 131072, "dtype": "bf16", "tokens": 1, "top": 1, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm; half of them as they fall, half round ones."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and x >= 64:
        x -= x % 32
    return max(lo, min(hi, x))


def draw(rng):
    op = rng.choice(("quantize", "dequantize", "norm", "matmul", "logprobs"))
    while True:
        if op in ("quantize", "dequantize"):
            case = {"op": op, "n": _log(rng, 1, 1_000_000), "d": _log(rng, 16, 8192), "dtype": rng.choice(("fp32", "bf16", "fp16")),
                    "format": rng.choice(("mxfp4", "mxfp8"))}
            if case["n"] * case["d"] * SIZE[case["dtype"]] <= 2_000_000_000:
                return case
        elif op == "norm":
            case = {"op": op, "n": _log(rng, 1, 8192), "d": _log(rng, 64, 8192), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                    "format": rng.choice(("mxfp8", "mxfp8", "mxfp4")), "residual": rng.random() < 0.75}
            if case["n"] * case["d"] * SIZE[case["dtype"]] <= 67_000_000:
                return case
        elif op == "matmul":
            case = {"op": op, "m": _log(rng, 1, 4096), "n": _log(rng, 16, 131072), "k": _log(rng, 64, 8192), "a": rng.choice(("mxfp8", "mxfp8", "mxfp4")),
                    "out": rng.choice(("fp32", "bf16"))}
            if case["m"] * case["n"] * case["k"] <= 1_000_000_000_000 and case["n"] * case["k"] <= 536_000_000 and case["m"] * case["n"] <= 260_000_000:
                return case
        else:
            case = {"op": op, "n": _log(rng, 1, 4096), "v": _log(rng, 1000, 262144), "dtype": rng.choice(("fp32", "bf16", "fp16")),
                    "tokens": rng.choice((1, 1, 2, 7)), "top": rng.choice((0, 1, 5, 20, 64)), "masked": rng.choice((0.0, 0.0, 0.3, 0.9))}
            if case["n"] * case["v"] * SIZE[case["dtype"]] <= 536_000_000:
                return case


def _padded(d):
    return -(-d // PAD) * PAD


def _power(s):
    """2^s in 32 bits, -127 <= s <= 127, put together from its bits (the lowest one is subnormal)."""
    bits = torch.where(s == -127, torch.full_like(s, 0x00400000), (s + 127) << 23)
    return bits.to(torch.int32).view(torch.float32)


def _quantized(x, fmt):
    """(element values, 2^s of each block, s with 128 for a block that holds no number) of 32-bit rows padded to whole blocks."""
    top, largest, up, bits = ELEMENT[fmt]
    y = x.reshape(x.shape[0], -1, BLOCK)
    a = y.abs().amax(dim=2)
    bad = ~torch.isfinite(a)
    a = torch.where(bad, torch.ones_like(a), a)
    s = torch.frexp(a).exponent.to(torch.int32) - 1 - top
    s = s.clamp(min=-127)
    r = a * _power(-s)
    s = s + ((r >= up) if fmt == "mxfp4" else (r > up)).to(torch.int32)
    s = torch.where(a == 0, torch.full_like(s, -127), s)
    y = y * _power(-s).unsqueeze(2)
    e = (torch.frexp(y).exponent.to(torch.int32) - 1).clamp(min=0 if fmt == "mxfp4" else -6)
    step = e - (bits - 1)
    q = torch.round(y * _power(-step)) * _power(step)
    q = q.clamp(-largest, largest)
    return torch.where(bad.unsqueeze(2), torch.zeros_like(q), q), _power(s), torch.where(bad, torch.full_like(s, 128), s)


def _values(q, scale, s, d):
    """What quantised rows stand for, 32 bits."""
    v = q * scale.unsqueeze(2)
    v = torch.where((s == 128).unsqueeze(2), torch.full_like(v, math.nan), v)
    return v.reshape(v.shape[0], -1)[:, :d]


def _packed(x, fmt):
    """Rows in their stored form: (element bytes, scale bytes)."""
    q, _, s = _quantized(_fill(x), fmt)
    q, scales = q.reshape(x.shape[0], -1), (s + 127).to(torch.uint8)
    if fmt == "mxfp8":
        return q.to(torch.float8_e4m3fn).view(torch.uint8), scales
    m = q.abs()
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m * 0.5 + 4)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scales


def _fill(x):
    x = x.float()
    more = _padded(x.shape[1]) - x.shape[1]
    return torch.nn.functional.pad(x, (0, more)) if more else x


def _unpacked(values, scales, fmt, d):
    """What stored rows stand for, 32 bits."""
    if fmt == "mxfp8":
        q = values.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=values.device)
        q = table[torch.stack((values & 15, values >> 4), dim=2).to(torch.int32)]
    s = scales.to(torch.int32) - 127
    return _values(q.reshape(values.shape[0], -1, BLOCK), _power(s.clamp(max=127)), s, d)


def _in_parts(n, d):
    """Row ranges of about a hundred million elements, so that making the inputs does not need many times their size."""
    rows = max(1, 100_000_000 // max(1, d))
    return [(r, min(n, r + rows)) for r in range(0, n, rows)]


def _rows(n, d, dtype, g):
    """Embedding-like rows: normal values, each row of a length of its own, a few columns much larger than the others."""
    scale = torch.exp(torch.randn(d, generator=g, device="cuda") * 0.5)
    out = torch.empty((n, d), dtype=dtype, device="cuda")
    for lo, hi in _in_parts(n, d):
        length = torch.exp(torch.randn(hi - lo, 1, generator=g, device="cuda"))
        out[lo:hi] = (torch.randn(hi - lo, d, generator=g, device="cuda") * scale * length).to(dtype)
    return out


def _stored(n, d, fmt, g):
    """Embedding-like rows in their stored form."""
    width = _padded(d)
    values = torch.empty((n, width // 2 if fmt == "mxfp4" else width), dtype=torch.uint8, device="cuda")
    scales = torch.empty((n, width // BLOCK), dtype=torch.uint8, device="cuda")
    for lo, hi in _in_parts(n, d):
        values[lo:hi], scales[lo:hi] = _packed(_rows(hi - lo, d, torch.float32, g), fmt)
    return values, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, state = case["op"], dict(case)
    if op == "quantize":
        state["x"] = _rows(case["n"], case["d"], DTYPES[case["dtype"]], g)
    elif op == "dequantize":
        state["x"] = _stored(case["n"], case["d"], case["format"], g)
    elif op == "norm":
        dtype = DTYPES[case["dtype"]]
        state["x"] = _rows(case["n"], case["d"], dtype, g)
        state["res"] = _rows(case["n"], case["d"], dtype, g) if case["residual"] else None
        state["w"] = (1 + 0.2 * torch.randn(case["d"], generator=g, device="cuda")).to(dtype)
    elif op == "matmul":
        state["A"] = _stored(case["m"], case["k"], case["a"], g)
        state["B"] = _stored(case["n"], case["k"], "mxfp4", g)
    else:
        n, v = case["n"], case["v"]
        logits = torch.empty((n, v), dtype=DTYPES[case["dtype"]], device="cuda")
        for lo, hi in _in_parts(n, v):
            part = torch.randn(hi - lo, v, generator=g, device="cuda") * (1 + 3 * torch.rand(hi - lo, 1, generator=g, device="cuda"))
            if case["masked"]:
                part.masked_fill_(torch.rand(hi - lo, v, generator=g, device="cuda") < case["masked"], -math.inf)
            logits[lo:hi] = part.to(logits.dtype)
        if n > 8:
            logits[n // 2] = -math.inf          # a row whose mask leaves nothing
        tokens = torch.randint(0, v, (n, case["tokens"]), generator=g, device="cuda")
        if n > 2:
            tokens[n // 3, -1] = -1             # padding: nothing is asked there
        state["logits"], state["tokens"] = logits, tokens
    return state


def run(state):
    op = state["op"]
    if own:
        from medical_rag_amd import scoring
        if op == "quantize":
            return scoring.mx_dequantize(scoring.mx_quantize(state["x"], state["format"]), torch.bfloat16)
        if op == "dequantize":
            return scoring.mx_dequantize(scoring.MxRows(*state["x"], state["d"], state["format"]), DTYPES[state["dtype"]])
        if op == "norm":
            y, h = scoring.rms_norm_mx(state["x"], state["w"], 1e-6, state["res"], state["format"])
            y = scoring.mx_dequantize(y, torch.bfloat16)
            return {"y": y, "h": h} if state["residual"] else {"y": y}
        if op == "matmul":
            return scoring.mx_matmul(scoring.MxRows(*state["A"], state["k"], state["a"]), scoring.MxRows(*state["B"], state["k"], "mxfp4"), DTYPES[state["out"]])
        r = scoring.token_logprobs(state["logits"], state["tokens"], state["top"])
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        return out | {"top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if state["top"] else out

    if op == "quantize":
        return _values(*_quantized(_fill(state["x"]), state["format"]), state["d"]).to(torch.bfloat16)
    if op == "dequantize":
        return _unpacked(*state["x"], state["format"], state["d"]).to(DTYPES[state["dtype"]])
    if op == "norm":
        h = state["x"]
        if state["residual"]:
            h = (h.float() + state["res"].float()).to(h.dtype)
        f = h.float()
        y = f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + 1e-6) * state["w"].float()
        y = _values(*_quantized(_fill(y), state["format"]), state["d"]).to(torch.bfloat16)
        return {"y": y, "h": h} if state["residual"] else {"y": y}
    if op == "matmul":
        a, b = _unpacked(*state["A"], state["a"], state["k"]), _unpacked(*state["B"], "mxfp4", state["k"])
        return (a @ b.t()).to(DTYPES[state["out"]])

    logits, tokens, top = state["logits"].float(), state["tokens"], state["top"]
    v = logits.shape[1]
    peak = logits.amax(dim=1, keepdim=True)
    peak = torch.where(torch.isinf(peak), torch.zeros_like(peak), peak)
    z = logits - peak
    p = torch.exp(z)
    total = p.sum(dim=1, keepdim=True)
    log_total = torch.log(total)
    lp = z.gather(1, tokens.clamp(0, v - 1)) - log_total
    lp = torch.where(total == 0, torch.full_like(lp, -math.inf), lp)
    lp = torch.where(tokens < 0, torch.zeros_like(lp), lp)
    entropy = log_total - torch.where(p > 0, p * z, torch.zeros_like(z)).sum(dim=1, keepdim=True) / total
    entropy = torch.where(total == 0, torch.zeros_like(entropy), entropy).squeeze(1)
    out = {"logprobs": lp, "entropy": entropy}
    if top:
        # one whole number for (logit, place), larger for the larger logit and then for the earlier place
        bits = (logits + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
        best = ((order << 32) + (v - 1 - torch.arange(v, device=logits.device))).topk(top, dim=1).values
        ids = v - 1 - (best & 0xFFFFFFFF)
        top_lp = z.gather(1, ids) - log_total
        gone = (logits.gather(1, ids) == -math.inf) | (total == 0)
        out["top_ids"] = torch.where(gone, torch.full_like(ids, -1), ids)
        out["top_logprobs"] = torch.where(gone, torch.full_like(top_lp, -math.inf), top_lp)
    return out


def work(case):
    op = case["op"]
    if op in ("quantize", "dequantize", "norm"):
        n, d = case["n"], case["d"]
        stored = n * (_padded(d) // (2 if case["format"] == "mxfp4" else 1) + _padded(d) // BLOCK)
        plain = n * d * SIZE[case["dtype"]]
        if op == "quantize":
            return {"bytes": plain + 2 * stored + n * d * 2, "flops": 4 * n * d}
        if op == "dequantize":
            return {"bytes": stored + plain, "flops": n * d}
        return {"bytes": plain * (3 if case["residual"] else 1) + d * SIZE[case["dtype"]] + 2 * stored + n * d * 2, "flops": 8 * n * d}
    if op == "matmul":
        m, n, k = case["m"], case["n"], _padded(case["k"])
        return {"bytes": m * (k // (2 if case["a"] == "mxfp4" else 1) + k // BLOCK) + n * (k // 2 + k // BLOCK) + m * n * SIZE[case["out"]],
                "flops": 2 * m * n * case["k"]}
    n, v = case["n"], case["v"]
    return {"bytes": n * v * SIZE[case["dtype"]] + n * (case["tokens"] * 12 + case["top"] * 12 + 4), "flops": 5 * n * v}


def _two_to(s):
    """2^s in 64 bits, from its exponent field (a device's pow may be off in its last bit, which moves ties)."""
    return ((s.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_quantized(x, fmt):
    """Rows in 64 bits: every value replaced by the nearest of the format's values in its block's scale, found in a list of them."""
    if fmt == "mxfp4":
        grid, largest_exponent = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], 2
    else:
        grid, largest_exponent = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1], 8
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    n, d = x.shape
    y = torch.zeros((n, -(-d // 32) * 32), dtype=torch.float64, device=x.device)
    y[:, :d] = x
    y = y.reshape(n, -1, 32)
    a = y.abs().max(dim=2, keepdim=True).values
    # the smallest power of two under which the block's largest value rounds to the list's largest or less
    tie = (grid[-1] + (grid[-1] * 2 - grid[-2])) / 2
    s = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))) - largest_exponent - 2
    for _ in range(4):
        r = a / _two_to(s)
        s = torch.where((r >= tie) if fmt == "mxfp4" else (r > tie), s + 1, s)
    s = torch.where(a > 0, s, torch.zeros_like(s)).clamp(min=-127)
    u = _two_to(s)
    m = (y / u).abs()
    above = torch.searchsorted(grid, m).clamp(max=grid.numel() - 1)     # the first value that is not smaller
    below = (above - 1).clamp(min=0)
    hi, lo = grid[above] - m, m - grid[below]
    m = grid[torch.where((lo < hi) | ((lo == hi) & (below % 2 == 0)), below, above)]
    return (torch.copysign(m, y) * u).reshape(n, -1)[:, :d]


def _exact_stored(values, scales, fmt, d):
    n = values.shape[0]
    if fmt == "mxfp4":
        grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        codes = torch.empty((n, values.shape[1] * 2), dtype=torch.int64, device=values.device)
        codes[:, 0::2], codes[:, 1::2] = values % 16, values // 16
    else:
        grid = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
        codes = values.to(torch.int64)
    table = torch.tensor(grid + [-v for v in grid], dtype=torch.float64, device=values.device)
    power = _two_to(scales.to(torch.int64) - 127)
    return (table[codes] * power.repeat_interleave(32, dim=1))[:, :d]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        out = torch.empty((case["n"], case["d"]), dtype=torch.float64, device="cuda")
        for lo, hi in _in_parts(case["n"], case["d"]):
            out[lo:hi] = _exact_quantized(state["x"][lo:hi].double(), case["format"])
        return out
    if op == "dequantize":
        out = torch.empty((case["n"], case["d"]), dtype=torch.float64, device="cuda")
        for lo, hi in _in_parts(case["n"], case["d"]):
            out[lo:hi] = _exact_stored(state["x"][0][lo:hi], state["x"][1][lo:hi], case["format"], case["d"])
        return out
    if op == "norm":
        h = state["x"].double()
        if case["residual"]:
            h = (h + state["res"].double()).to(state["x"].dtype).double()
        y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["d"] + 1e-6) * state["w"].double()
        y = _exact_quantized(y, case["format"])
        return {"y": y, "h": h} if case["residual"] else {"y": y}
    if op == "matmul":
        a = _exact_stored(*state["A"], case["a"], case["k"])
        out = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for lo, hi in _in_parts(case["n"], case["k"]):
            out[:, lo:hi] = a @ _exact_stored(state["B"][0][lo:hi], state["B"][1][lo:hi], "mxfp4", case["k"]).t()
        return out
    parts = []
    for lo, hi in _in_parts(case["n"], case["v"]):
        logits, tokens = state["logits"][lo:hi].double(), state["tokens"][lo:hi]
        lse = torch.logsumexp(logits, dim=1, keepdim=True)
        empty = torch.isinf(lse)
        logp = torch.where(empty, torch.full_like(logits, -math.inf), logits - lse)
        entropy = -torch.special.xlogy(logp.exp(), logp.exp()).sum(dim=1)
        asked = torch.where(tokens < 0, torch.zeros((), dtype=torch.float64, device="cuda"), logp.gather(1, tokens.clamp(min=0)))
        part = {"logprobs": asked, "entropy": entropy}
        if case["top"]:
            got = torch.sort(logits, dim=1, descending=True, stable=True)
            ids, vals = got.indices[:, : case["top"]], got.values[:, : case["top"]]
            part["top_ids"] = torch.where(vals == -math.inf, torch.full_like(ids, -1), ids)
            part["top_logprobs"] = torch.where(empty, torch.full_like(vals, -math.inf), vals - lse)
        parts.append(part)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
