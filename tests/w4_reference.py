"""Weights in 4 bits and log probabilities in plain 64-bit numpy, from their definitions. Values are f64, bf16 arrays are
bit patterns (uint16)."""
import numpy as np

from common import bf16_bits, bf16_vals

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([GRID, -GRID])
LEAST = 2.0 ** -126
NONE = 0xFFFFFFFF


def bits(x):
    return np.asarray(bf16_bits(np.asarray(x, np.float32))).reshape(np.shape(x))


def vals(b):
    return np.asarray(bf16_vals(np.asarray(b, np.uint16)), np.float64).reshape(np.shape(b))


def whole(x, fill=0.0):
    """Rows and columns up to whole tiles."""
    r, c = x.shape
    out = np.full((-(-r // 16) * 16, -(-c // 128) * 128), fill, x.dtype)
    out[:r, :c] = x
    return out


def quantise(w, group):
    """Codes and scales (f64) of w [rows][cols] (f64 holding bf16 values), whole tiles of both."""
    x = whole(w).reshape(-1, -(-w.shape[1] // 128) * 128 // group, group)
    fin = np.isfinite(x).all(-1, keepdims=True)
    top = np.abs(np.where(fin, x, 0.0)).max(-1, keepdims=True) / 6.0
    _, e = np.frexp(top)
    unit = 2.0 ** (e - 8.0)
    s = np.maximum(np.where(top > 0, np.round(top / unit) * unit, 0.0), LEAST)
    q = np.abs(np.where(fin, x, 0.0)) / s  # exact where it matters: at the middles of two codes
    hi = np.clip(np.searchsorted(GRID, q), 1, 7)
    down, up = q - GRID[hi - 1], GRID[hi] - q
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    code = code + 8 * (np.signbit(x) & fin)
    return code.reshape(-1, x.shape[1] * group), np.where(fin, s, np.nan)[..., 0]


def lay(code, s):
    """The bytes of codes and scales (bf16 bits) of whole tiles, element by element from where they lie."""
    rows, cols = code.shape
    group = cols // s.shape[1]
    r, c = np.indices(code.shape)
    tile, k = r // 16 * (cols // 128) + c // 128, c % 128
    at = tile * 1024 + k // 8 % 4 * 256 + r % 16 * 16 + k // 32 * 4 + k % 8 // 2
    codes = np.zeros(rows * cols // 2, np.uint8)
    np.add.at(codes, at.ravel(), (code * np.where(k % 2, 16, 1)).astype(np.uint8).ravel())
    r, g = np.indices(s.shape)
    per = 128 // group
    scales = np.zeros(s.size, np.uint16)
    scales[((r // 16 * (cols // 128) + g // per) * 16 + r % 16) * per + g % per] = bits(s)
    return codes, scales


def values(code, s):
    """What codes and scales stand for."""
    return VALUES[code] * np.repeat(s, code.shape[1] // s.shape[1], 1)


def logprobs(x, scale, tokens=None, top=0):
    """(token_lp, entropy, top_ids, top_lp) of rows x (f64 holding the logits)."""
    rows, vocab = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        y = x * float(np.float32(scale))
        m = y.max(-1, keepdims=True)
        ok = np.isfinite(y.sum(-1)) | (np.isfinite(m[:, 0]) & ~np.isnan(y).any(-1))
        p = np.exp(y - m)
        z = p.sum(-1, keepdims=True)
        lp = np.where(ok[:, None], y - m - np.log(z), np.nan)
        entropy = np.where(ok, (np.log(z) - np.where(p > 0, p * (y - m), 0.0).sum(-1, keepdims=True) / z)[:, 0], np.nan)
    ids, best = np.full((rows, top), NONE, np.uint32), np.full((rows, top), -np.inf)
    best[~ok] = np.nan
    for r in np.nonzero(ok)[0]:
        order = np.lexsort((np.arange(vocab), -x[r]))
        order = order[x[r][order] > -np.inf][:top]
        ids[r, :len(order)], best[r, :len(order)] = order, lp[r, order]
    token_lp = None
    if tokens is not None:
        known = tokens < vocab
        token_lp = np.where(known, np.take_along_axis(lp, np.where(known, tokens, 0).astype(np.int64), 1), np.nan)
    return token_lp, entropy, ids, best
