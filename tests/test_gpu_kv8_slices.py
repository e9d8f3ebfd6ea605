"""Decode attention over the 8-bit paged K/V cache where blocks walk several slices: batches whose blocks count and join
slices while they hold further ones (tests/test_cpu_kv8_slices.py holds the shapes to that)."""
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
