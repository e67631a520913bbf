"""The scoring head's operators in numpy float64, from their definitions: test
infrastructure only.

Microscaled rows are kept as (codes, scales): codes (n, padded d) uint8, one
element a byte whatever the format, scales (n, padded d / 32) uint8."""
import numpy as np

BLOCK, PAD = 32, 128
GRID = {"mxfp4": np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]),
        "mxfp8": np.array([m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])}
LARGEST_EXPONENT = {"mxfp4": 2, "mxfp8": 8}


def padded(d):
    return -(-d // PAD) * PAD


def mx_scale(a, fmt):
    """The scale's exponent for blocks of largest magnitude a (finite): the smallest
    power of two, not below 2^-127, under which a rounds to the largest element or
    less.  7 would round to 8 (even) and does not fit, 464 to 448 (even) and does."""
    _, e = np.frexp(a)
    s = np.maximum(e - 1 - LARGEST_EXPONENT[fmt], -127)
    r = np.ldexp(a, -s)
    s = s + ((r >= 7.0) if fmt == "mxfp4" else (r > 464.0))
    return np.where(a == 0, -127, s)


def mx_quantize(x, fmt):
    """(codes, scales) of rows x."""
    x = np.asarray(x, dtype=np.float64)
    n, d = x.shape
    y = np.zeros((n, padded(d)))
    y[:, :d] = x
    y = y.reshape(n, padded(d) // BLOCK, BLOCK)
    bad = ~np.isfinite(y).all(axis=2)
    y = np.where(bad[:, :, None], 0.0, y)
    s = mx_scale(np.abs(y).max(axis=2), fmt)
    m = np.ldexp(np.abs(y), -s[:, :, None])
    grid = GRID[fmt]
    above = np.minimum(np.searchsorted(grid, m), len(grid) - 1)
    below = np.maximum(above - 1, 0)
    hi, lo = grid[above] - m, m - grid[below]
    code = np.where((lo < hi) | ((lo == hi) & (below % 2 == 0)), below, above)
    sign = np.signbit(y) * (8 if fmt == "mxfp4" else 128)
    codes = np.where(bad[:, :, None], 0, code + sign).astype(np.uint8)
    return codes.reshape(n, padded(d)), np.where(bad, 255, s + 127).astype(np.uint8)


def mx_values(codes, scales, fmt, d):
    """What (codes, scales) stand for, float64 (n, d)."""
    grid = GRID[fmt]
    if fmt == "mxfp8":
        grid = np.concatenate([grid, [np.nan]])
    table = np.concatenate([grid, -grid])
    v = table[codes].reshape(codes.shape[0], codes.shape[1] // BLOCK, BLOCK)
    s = scales.astype(np.int64) - 127
    with np.errstate(invalid="ignore"):
        v = np.where((scales == 255)[:, :, None], np.nan, np.ldexp(v, np.where(scales == 255, 0, s)[:, :, None]))
    return v.reshape(codes.shape)[:, :d]


def pack(codes, fmt):
    """Codes as stored: two 4-bit elements a byte, the earlier one in the low half."""
    return codes if fmt == "mxfp8" else (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(values, fmt):
    if fmt == "mxfp8":
        return values
    out = np.empty((values.shape[0], values.shape[1] * 2), np.uint8)
    out[:, 0::2], out[:, 1::2] = values & 15, values >> 4
    return out


def rms_norm(h, weight, eps):
    h = np.asarray(h, np.float64)
    return h / np.sqrt((h * h).sum(axis=1, keepdims=True) / h.shape[1] + eps) * np.asarray(weight, np.float64)


def token_logprobs(logits, tokens, top_k):
    """(logprobs, entropy, top ids, top log probabilities) by the definitions of
    include/medtutor_retrieval.h."""
    logits, tokens = np.asarray(logits, np.float64), np.asarray(tokens, np.int64)
    n, v = logits.shape
    lp, entropy = np.zeros(tokens.shape), np.zeros(n)
    ids, tlp = np.full((n, top_k), -1, np.int64), np.full((n, top_k), -np.inf)
    for i in range(n):
        row = logits[i]
        if np.isnan(row).any() or (row == np.inf).any():
            lp[i], entropy[i], tlp[i] = np.nan, np.nan, np.nan
        else:
            left = row > -np.inf
            logp = np.full(v, -np.inf)
            if left.any():
                m = row.max()
                logp[left] = (row[left] - m) - np.log(np.exp(row[left] - m).sum())
                entropy[i] = -(np.exp(logp[left]) * logp[left]).sum()
            order = np.argsort(-row, kind="stable")[: min(top_k, int(left.sum()))]
            ids[i, : len(order)], tlp[i, : len(order)] = order, logp[order]
            inside = (tokens[i] >= 0) & (tokens[i] < v)
            lp[i] = np.where(inside, logp[np.where(inside, tokens[i], 0)], 0.0)
        lp[i][tokens[i] >= v] = np.nan
        lp[i][tokens[i] < 0] = 0.0
    return lp, entropy, ids, tlp
