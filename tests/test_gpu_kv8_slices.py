"""Decode attention over the 8-bit paged K/V cache where blocks walk several slices, with outputs that show every page
and key: batches whose blocks count and join slices while they hold further ones (tests/test_cpu_kv8_slices.py holds
the shapes to that), a scale of 0 over values that count keys, and flat scores within a bound in which a single
page stands out."""
import numpy as np
import pytest

import kv8_reference as R
from kv8_reference import HEAD, NONE, PAGE, bits, vals
from test_gpu_kv8 import check_attention, random_q

pytestmark = pytest.mark.gpu

# (group, kv heads, the lengths of four kinds of sequence, sequences, pages of a table, budget): the kinds in turn.
WALKS = [
    (2, 8, [2000, 1990, 1951, 2000], 40, 126, 0),
    (5, 8, [6000, 6000, 5900, 60], 20, 376, 0),
    # More loads than the Infinity Cache holds, at each number of parts of a join by 8 wavefronts.
    (1, 8, [6000, 5500, 6000, 5999], 40, 376, 0),
    (8, 8, [6000, 5500, 6000, 5999], 40, 376, 0),
    (12, 8, [6000, 5500, 6000, 5999], 40, 376, 0),
    # Blocks of 4 wavefronts, at each number of parts of their joins.
    (2, 2, [2000, 1990, 1951, 2000], 40, 126, 0),
    (4, 2, [2000, 1990, 1951, 2000], 40, 126, 0),
    (8, 2, [2000, 1990, 1951, 2000], 40, 126, 0),
    (16, 2, [2000, 1990, 1951, 2000], 40, 126, 0),
    # Uneven ones, a list's pages, more than 64 sequences.
    (16, 2, [6000, 6000, 5900, 60], 40, 376, 0),
    (3, 4, [4700, 4800, 17, 4000], 32, 300, 0),
    (4, 8, [6000, 5500, 6000, 5999], 40, 376, 200),
    (4, 2, [2000, 1990, 1951, 2000], 70, 126, 0),
]


def pooled(rng, kv_heads, kinds, seqs, seq_pages, pool=96):
    """Sequences of a few kinds over a small pool of random pages: kind i's table, shared by sequences i, i + 4, ..."""
    c = R.fill(rng, kv_heads, [pool * PAGE], pool, spare=0)
    tables = rng.integers(0, pool, (len(kinds), seq_pages)).astype(np.uint32)
    of = np.arange(seqs) % len(kinds)
    return type(c)(c.codes, c.scales, tables[of]), of


def kinds_only(c, n):
    return type(c)(c.codes, c.scales, c.table[:n])


@pytest.mark.parametrize("group,kv_heads,kinds,seqs,seq_pages,budget", WALKS)
def test_attention_of_blocks_that_walk_slices(kernels, group, kv_heads, kinds, seqs, seq_pages, budget):
    """Sequences of one kind have one output, bit for bit, wherever their slices lie and whichever block joins them, in
    every call over one workspace; the kinds' outputs are those of the plain form."""
    rng = np.random.default_rng(group * 1000 + kv_heads * 100 + seqs)
    c, of = pooled(rng, kv_heads, kinds, seqs, seq_pages)
    n, q_heads = len(kinds), group * kv_heads
    q = random_q(rng, n, q_heads)
    pages = None
    if budget:
        pages = np.full((n, kv_heads, budget), NONE, np.uint32)
        for s in range(n):
            for h in range(kv_heads):
                pages[s, h] = np.sort(rng.permutation(-(-kinds[s] // PAGE))[:budget])
    lens = np.array(kinds)[of]
    for calls in (1, 3):
        out = kernels.kv8_attention(c, q[of], q_heads, lens, page_list=None if pages is None else pages[of], calls=calls)
        assert (out == out[:n][of]).all(), "sequences of one kind differ"
    check_attention(kinds_only(c, n), q, q_heads, kinds, out[:n], page_list=pages)


# -- values that count keys --

# (group, kv heads, lengths, pages of a table)
COUNTED = [
    (4, 2, [20000], 1259),
    (1, 1, [4097, 64, 65, 63, 1], 270),
    (3, 2, [9000, 8191, 8192, 8193], 572),
    (7, 1, [n for m in range(1, 33) for n in (64 * m - 1, 64 * m, 64 * m + 1)][:62], 128),
    (2, 8, [2000, 1990, 1951, 2000] * 10, 126),
    (2, 2, [2000, 1985, 1984, 1983] * 10, 126),
    (8, 8, [6000, 5500, 6000, 5999] * 10, 376),
    (5, 8, [6000, 6000, 5900, 60] * 5, 376),
    (1, 4, [4700, 4800, 17, 4000] * 8, 300),
    (1, 8, [16384, 777, 40] + [33] * 5, 1100),
]
COUNT_OFF = 2.0 ** -8 + 2.0 ** -21  # the rounding to bf16 and, in f32, of 1 / n and its product: a few 2^-24


def counting(rng, kv_heads, lens, seq_pages):
    """A cache of 128 pages whose values are 1 in one dim and 0 in the others: dim (a_h p + b_h) % 127 in page p < 127,
    so that each kv head deals the pages to its dims in its own order, and 127 in page 127. Tables use the first 127 pages
    about as often, and 127 for every sequence's last: (cache, dim of each page [kv_heads][128])."""
    page = np.arange(128)
    a, b = rng.integers(1, 127, (2, kv_heads))
    dims = np.where(page < 127, (a[:, None] * page + b[:, None]) % 127, 127)
    v = np.zeros((128, kv_heads, PAGE, HEAD))
    for h in range(kv_heads):
        v[page, h, :, dims[h]] = 1.0
    c = R.fill(rng, kv_heads, [128 * PAGE], 128, spare=0)
    vc, vs = R.quantise(v)
    c.codes[:, :, 2048:] = vc.transpose(0, 1, 3, 2).reshape(128, kv_heads, 2048)
    c.scales[:, :, PAGE:] = vs
    table = np.stack([np.concatenate([rng.permutation(127) for _ in range(-(-seq_pages // 127))])[:seq_pages] for _ in lens])
    for s, n in enumerate(lens):
        table[s, -(-n // PAGE) - 1] = 127
    return type(c)(c.codes, c.scales, table.astype(np.uint32)), dims


def counts(c, dims, s, n):
    """Keys of sequence s below n in each dim, [kv_heads][128], and of each of its pages: [pages]."""
    keys = np.minimum(PAGE, n - PAGE * np.arange(-(-n // PAGE)))
    at = dims[:, c.table[s, :len(keys)]]
    return np.stack([np.bincount(at[h], keys, HEAD) for h in range(len(dims))]), keys


@pytest.mark.parametrize("group,kv_heads,lens,seq_pages", COUNTED)
def test_every_page_and_key_counts_once(kernels, group, kv_heads, lens, seq_pages):
    """At a scale of 0 every key weighs 1 and the sums are whole numbers, exact in f32: an output is its dim's keys over
    the sequence's, within the final roundings. A page left out, taken twice or for another moves some dim by more, and
    so does a key of the last page or one behind the length."""
    rng = np.random.default_rng(len(lens) * 100 + kv_heads)
    c, dims = counting(rng, kv_heads, lens, seq_pages)
    q = random_q(rng, len(lens), group * kv_heads)
    out = vals(kernels.kv8_attention(c, q, group * kv_heads, lens, scale=0.0, calls=2)).reshape(len(lens), kv_heads, group, HEAD)
    for s, n in enumerate(lens):
        want = counts(c, dims, s, n)[0][:, None] / n
        assert (np.abs(out[s] - want) <= COUNT_OFF * want).all(), f"sequence {s} of {n} keys"


# -- flat scores --

# (group, kv heads, lengths, pages of a table, the most tiles a wavefront takes of a slice)
FLAT = [
    (4, 2, [20000], 1259, 2),
    (4, 2, [9000, 8191], 572, 1),
    (8, 1, [4097, 1025], 270, 1),
    (4, 8, [6000, 5500, 6000, 5999] * 10, 376, 6),
    (2, 2, [2000, 1990, 1951, 2000] * 10, 126, 1),
]
FLAT_Q = 0.1


def flat_tolerance(keys_v, weights, q, k, scale, rounds):
    """How far the outputs of one kv head [group][128] may be from their 64-bit values, by the kernel's steps. A score in
    units of log 2 is a sum of 128 exact products in f32 in any order (130 roundings), times a factor of three roundings
    and less a maximum (two more, of numbers up to the largest score twice): its weight is off by ln 2 times that. Each
    of a wavefront's `rounds` tiles may rescale what is before it, as do the joins of wavefronts and of slices: an exponential
    (1 ulp, 2^-23) and a product each. A weight is two bf16 parts (2^-17 of it). The value sums round at most 33 times a
    matrix instruction, 4 of which a dim's sum takes of each tile (2 by 32 keys, of both parts), and once per wavefront
    and slice (8 + 64); the sum of the weights 16 times a tile and once per lane, wavefront and slice. Those go with the sum of
    |v| under the weights; what the denominator has, with the output; then a division and a product, and the rounding
    to bf16."""
    reach = float((np.abs(q) @ np.abs(k).T).max()) * abs(scale) * np.log2(np.e)
    share = weights / weights.sum(-1, keepdims=True)
    spread, want = share @ np.abs(keys_v), share @ keys_v
    weight = np.log(2) * 135 * 2.0 ** -24 * reach + (rounds + 3) * 3 * 2.0 ** -23
    return (spread * (weight + 2.0 ** -17 + (132 * rounds + 80) * 2.0 ** -24)
            + np.abs(want) * (weight + (16 * rounds + 80) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -8))


def flat_case(group, kv_heads, lens, seq_pages):
    """(cache, queries, number of kinds): random keys and values, every page of a sequence another of the pool."""
    rng = np.random.default_rng(len(lens) * 10 + group)
    n = min(len(lens), 4)
    c = R.fill(rng, kv_heads, [seq_pages * PAGE], seq_pages, spare=0)
    tables = np.stack([rng.permutation(seq_pages) for _ in range(n)]).astype(np.uint32)
    return type(c)(c.codes, c.scales, tables), random_q(rng, n, group * kv_heads, FLAT_Q), n


def flat_weights(c, q, s, h, n, scale):
    """Of kv head h of sequence s: keys, values [n][128], the weights [group][n]."""
    k, v = (x[h] for x in R.sequence(c, s, n))
    x = q @ k.T * scale
    return k, v, np.exp(x - x.max(-1, keepdims=True))


@pytest.mark.parametrize("group,kv_heads,lens,seq_pages,rounds", FLAT)
def test_attention_of_flat_scores_misses_no_page(kernels, group, kv_heads, lens, seq_pages, rounds):
    from x0ne_core.ops import attn_scale
    c, q, n = flat_case(group, kv_heads, lens, seq_pages)
    of, scale = np.arange(len(lens)) % n, attn_scale(HEAD)
    out = kernels.kv8_attention(type(c)(c.codes, c.scales, c.table[of]), q[of], group * kv_heads, lens, calls=2)
    assert (out == out[:n][of]).all()
    got, qv, worst = vals(out[:n]).reshape(n, kv_heads, group, HEAD), vals(q).reshape(n, kv_heads, group, HEAD), 0.0
    for s in range(n):
        for h in range(kv_heads):
            k, v, w = flat_weights(c, qv[s, h], s, h, lens[s], scale)
            tol = flat_tolerance(v, w, qv[s, h], k, scale, rounds)
            off = np.abs(got[s, h] - w @ v / w.sum(-1, keepdims=True))
            worst = max(worst, float((off / tol).max()))
            assert (off <= tol).all(), f"sequence {s} of {lens[s]} keys, kv head {h}: {(off / tol).max()} of the tolerance"
    print(f"MEASURE kv8 attention, flat scores {group}/{kv_heads} {lens[:4]}: worst {worst:.3f} of the tolerance")


# -- values of every size --

@pytest.mark.parametrize("power", [-124, -112, -100, 60, 115, None])
def test_attention_of_tiny_and_large_values(kernels, power):
    """Values around 2^power, and rows of sizes from 2^-40 to 2^40 beside each other (None), under ordinary scores:
    within flat_tolerance's bound. A weight times its row's power of two lies below bf16's normal numbers for tiny
    rows, where its second part is off by up to 2^-134 of the row's code, as is the output's own rounding."""
    from x0ne_core.ops import attn_scale
    rng = np.random.default_rng(200 + (power or 0))
    lens, kv_heads, group = [300, 40, 1, 700], 2, 4
    c = R.fill(rng, kv_heads, lens, 44)
    x = rng.standard_normal((c.pool, kv_heads, PAGE, HEAD))
    x *= 2.0 ** (power if power is not None else rng.integers(-40, 41, (c.pool, kv_heads, PAGE, 1)))
    vc, vs = R.quantise(vals(bits(x)).reshape(x.shape))
    c.codes[:, :, 2048:] = vc.transpose(0, 1, 3, 2).reshape(c.pool, kv_heads, 2048)
    c.scales[:, :, PAGE:] = vs
    q, scale = random_q(rng, len(lens), group * kv_heads), attn_scale(HEAD)
    got = vals(kernels.kv8_attention(c, q, group * kv_heads, lens)).reshape(len(lens), kv_heads, group, HEAD)
    qv, worst = vals(q).reshape(len(lens), kv_heads, group, HEAD), 0.0
    for s, n in enumerate(lens):
        page = c.table[s, np.arange(n) // PAGE]
        for h in range(kv_heads):
            k, v, w = flat_weights(c, qv[s, h], s, h, n, scale)
            e = R.powers(c.scales[page, h, PAGE + np.arange(n) % PAGE])[:, None]
            tol = flat_tolerance(v, w, qv[s, h], k, scale, 1) + 2.0 ** -134 * (1 + (np.abs(v) / e).sum(0) / w.sum(-1, keepdims=True))
            off = np.abs(got[s, h] - w @ v / w.sum(-1, keepdims=True))
            worst = max(worst, float((off / tol).max()))
            assert (off <= tol).all(), f"sequence {s} of {n} keys, kv head {h}: {(off / tol).max()} of the tolerance"
    print(f"MEASURE kv8 attention, values around 2^{power}: worst {worst:.3f} of the tolerance")
