"""The 8-bit paged K/V cache in plain 64-bit numpy, from its definition: rounding, layout, write, read-back,
attention, page scores. Values are f64, bf16 arrays are bit patterns (uint16)."""
import math

import numpy as np

from common import bf16_bits, bf16_vals

HEAD, PAGE, LOWEST, NONE = 128, 16, -117, 0xFFFFFFFF
GRID = np.array([c * 2.0 ** -9 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(127)])
VALUES = np.concatenate([GRID, [np.nan], -GRID, [np.nan]])  # of every code


def bits(x):
    return bf16_bits(np.asarray(x, np.float32))


def vals(b):
    return np.asarray(bf16_vals(np.asarray(b, np.uint16)), np.float64).reshape(np.shape(b))


def quantise(x):
    """Codes and scale bytes of rows x [..., 128] (f64 holding bf16 values)."""
    fin = np.isfinite(x)
    top = np.abs(np.where(fin, x, 0.0)).max(-1)
    m, e = np.frexp(top / 448.0)  # top / 448 = m 2^e, m in [0.5, 1): 2^e is above it, 2^(e - 1) equal to it at m = 0.5
    e = np.where(top == 0, LOWEST, np.where(m == 0.5, e - 1, e))
    # top / 448 is rounded: settle the exponent on the exact products
    e = np.where(448.0 * 2.0 ** (e - 1.0) >= top, e - 1, np.where(448.0 * 2.0 ** (1.0 * e) < top, e + 1, e))
    e = np.maximum(e, LOWEST).astype(np.int64)
    y = np.where(fin, x, 0.0) / 2.0 ** e[..., None].astype(np.float64)
    a = np.abs(y)
    hi = np.clip(np.searchsorted(GRID, a), 1, 126)
    down, up = a - GRID[hi - 1], GRID[hi] - a
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1) + np.where(np.signbit(y), 128, 0)
    return np.where(fin, code, 0x7F).astype(np.uint8), (e + 127).astype(np.uint8)


def powers(b):
    return 2.0 ** (b.astype(np.float64) - 127)


def empty(pool, kv_heads, seqs, seq_pages, rng=None, spare=0):
    """A cache of garbage: NaN codes and the largest scale bytes in every slot; the table a permutation."""
    from x0ne_core.ops import Kv8Pages
    order = np.arange(pool) if rng is None else rng.permutation(pool)
    return Kv8Pages(np.full((pool, kv_heads, 4096), 0x7F, np.uint8), np.full((pool, kv_heads, 32), 0xFF, np.uint8),
                    order[:seqs * seq_pages].reshape(seqs, seq_pages).astype(np.uint32))


def put(c, seq, pos, k, v):
    """Row (k, v) [kv_heads][128] f64 of bf16 values at position pos of sequence seq."""
    page = int(c.table[seq, pos // PAGE])
    if page >= c.pool:
        return
    slot = pos % PAGE
    for part, x in ((0, k), (1, v)):
        code, scale = quantise(x)
        if part == 0:
            c.codes[page, :, slot * HEAD:(slot + 1) * HEAD] = code
        else:
            c.codes[page, :, 2048 + slot::PAGE] = code
        c.scales[page, :, part * PAGE + slot] = scale


def fill(rng, kv_heads, lens, seq_pages, spare=3, drift=0.0):
    """A cache whose sequences hold random rows below lens (garbage elsewhere), pages shuffled among spare ones."""
    c = empty(len(lens) * seq_pages + spare, kv_heads, len(lens), seq_pages, rng)
    for s, n in enumerate(lens):
        n = min(n, seq_pages * PAGE)
        if n == 0:
            continue
        pages = -(-n // PAGE)
        kv = rng.standard_normal((2, pages * PAGE, kv_heads, HEAD))
        if drift:
            kv[0] += drift * np.repeat(rng.standard_normal((pages, kv_heads, HEAD)) * (rng.random((1, kv_heads, HEAD)) < 0.1),
                                       PAGE, 0)
        x = vals(bits(kv))
        kc, ks = quantise(x[0])
        vc, vs = quantise(x[1])
        kc[n:], vc[n:], ks[n:], vs[n:] = 0x7F, 0x7F, 0xFF, 0xFF
        at = c.table[s, :pages]
        split = lambda a: a.reshape(pages, PAGE, kv_heads, *a.shape[2:])
        c.codes[at, :, :2048] = split(kc).transpose(0, 2, 1, 3).reshape(pages, kv_heads, 2048)
        c.codes[at, :, 2048:] = split(vc).transpose(0, 2, 3, 1).reshape(pages, kv_heads, 2048)
        c.scales[at, :, :PAGE] = split(ks).transpose(0, 2, 1)
        c.scales[at, :, PAGE:] = split(vs).transpose(0, 2, 1)
    return c


def page_values(c, page):
    """K [kv_heads][16][128] and V [kv_heads][16][128] of a physical page."""
    with np.errstate(over="ignore", invalid="ignore"):
        k = VALUES[c.codes[page, :, :2048]].reshape(-1, PAGE, HEAD) * powers(c.scales[page, :, :PAGE])[..., None]
        v = VALUES[c.codes[page, :, 2048:]].reshape(-1, HEAD, PAGE) * powers(c.scales[page, :, PAGE:])[:, None]
    return k, v.transpose(0, 2, 1)


def sequence(c, seq, n, pages=None):
    """K, V [kv_heads][keys][128] of sequence seq's keys below n, of the pages in the table's pool only (pages: of
    those logical pages only)."""
    n = min(n, c.table.shape[1] * PAGE)
    ks, vs = [], []
    for p in range(-(-n // PAGE)) if pages is None else pages:
        at = int(c.table[seq, p])
        if at < c.pool:
            k, v = page_values(c, at)
            m = min(PAGE, n - p * PAGE)
            ks.append(k[:, :m])
            vs.append(v[:, :m])
    if not ks:
        return np.zeros((c.kv_heads, 0, HEAD)), np.zeros((c.kv_heads, 0, HEAD))
    return np.concatenate(ks, 1), np.concatenate(vs, 1)


def attention(q, k, v, scale):
    """One kv head: q [group][128], k, v [keys][128] -> (out [group][128], the weights' sums of |q k|: the largest
    over the keys, for the tolerance)."""
    if k.shape[0] == 0:
        return np.zeros_like(q), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        s = q @ k.T * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        return (p / p.sum(-1, keepdims=True)) @ v, float(np.nanmax(np.abs(q) @ np.abs(k).T) * abs(scale))


def bounds_of(c, page):
    """[kv_heads][2][128] bf16 bits of a complete page."""
    k, _ = page_values(c, page)
    with np.errstate(invalid="ignore"):
        b = np.stack([k.min(1), k.max(1)], 1) + 0.0  # numpy's min and max pass a NaN on; zeros are +0
    return np.where(np.isnan(b), 0x7FC0, bits(np.where(np.isnan(b), 0.0, b)).reshape(b.shape)).astype(np.uint16)


def all_bounds(c):
    return np.stack([bounds_of(c, p) for p in range(c.pool)])


def select(c, bounds, q, lens, budget):
    """The page list [seqs][kv_heads][budget]; q [seqs][q_heads][128] f64."""
    seqs, kvh = c.table.shape[0], c.kv_heads
    out = np.full((seqs, kvh, budget), NONE, np.uint32)
    b = vals(bounds)
    for s in range(seqs):
        n = -(-min(int(lens[s]), c.table.shape[1] * PAGE) // PAGE)
        for h in range(kvh):
            qs = q[s].reshape(kvh, -1, HEAD)[h]
            score = np.full(n, -math.inf)
            missing = np.ones(n, bool)
            for p in range(n):
                at = int(c.table[s, p])
                if at < c.pool:
                    missing[p] = False
                    with np.errstate(invalid="ignore"):
                        per = np.where(qs < 0, qs * b[at, h, 0], qs * b[at, h, 1]).sum(-1)
                    score[p] = np.nan if np.isnan(per).any() else per.max()
            # the last page, then NaN, then by score; the lower page first; a missing page last
            rank = sorted(range(n), key=lambda p: (p != n - 1, missing[p], not np.isnan(score[p]),
                                                   0.0 if np.isnan(score[p]) else -score[p], p))[:budget]
            out[s, h, :len(rank)] = sorted(rank)
    return out


def rotated(x, w, pos, theta, eps):
    """bf16 bits of RMSNorm (weights w) and RoPE at pos of heads x [heads][128] (f64)."""
    from x0ne_core.ops import inv_freq
    scale = 1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / HEAD + float(np.float32(eps)))
    n = x * scale * w
    angle = (np.float32(pos) * inv_freq(HEAD, theta)).astype(np.float64)
    a, b, co, si = n[:, :64], n[:, 64:], np.cos(angle), np.sin(angle)
    return bits(np.concatenate([a * co - b * si, b * co + a * si], 1)).reshape(x.shape)
