"""Calls of the 8-bit paged K/V cache at the ends of what they take: the widest tables, lengths past them in a selection,
query heads that are no multiple of the kv heads in a write, an output in the queries' place, pages that sequences share."""
import numpy as np
import pytest

import kv8_reference as R
from kv8_reference import HEAD, NONE, PAGE, vals
from test_gpu_kv8 import check_attention, check_read, check_write, random_q, random_qkv, widened
from test_gpu_kv8_slices import kinds_only, pooled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_heads,kv_heads", [(5, 2), (1, 8), (3, 4), (129, 3)])
def test_write_of_query_heads_that_are_no_multiple_of_the_kv_heads(kernels, q_heads, kv_heads):
    rng = np.random.default_rng(q_heads)
    row_seq, row_pos = [0] * 20 + [1, NONE, 2], list(range(10, 30)) + [15, 0, 31]
    check_write(kernels, rng, q_heads, kv_heads, random_qkv(rng, 23, q_heads, kv_heads), row_seq, row_pos, 2, 3)


def test_the_widest_tables(kernels):
    """2^24 - 1 pages to a sequence, of which it uses a few: write, read, attention; 65535 x 64 for the selection."""
    rng = np.random.default_rng(30)
    lens = [700]
    c = R.fill(rng, 1, lens, 44)
    wide = widened(c, (1 << 24) - 1)
    q = random_q(rng, 1, 4)
    check_attention(c, q, 4, lens, kernels.kv8_attention(wide, q, 4, lens, calls=2))
    out_table = np.full(wide.table.shape, NONE, np.uint32)
    out_table[0, :44] = rng.permutation(50)[:44]
    k, v = kernels.kv8_read(wide, lens, out_table, 50)
    check_read(kernels, c, lens, out_table, k, v)
    b = R.all_bounds(c)
    for budget in (1, 7, 60):
        got = kernels.kv8_select(widened(c, 65535 * 64), b, q, 4, lens, budget, calls=2)
        assert (got == R.select(c, b, vals(q), lens, budget)).all(), budget


@pytest.mark.parametrize("seq_pages", [3, 64, 65, 130])
def test_a_selection_clamps_lengths_to_the_table(kernels, seq_pages):
    rng = np.random.default_rng(seq_pages)
    room = seq_pages * PAGE
    c = R.fill(rng, 2, [room] * 3, seq_pages, drift=2.0)
    b, q = R.all_bounds(c), random_q(rng, 3, 6)
    want = R.select(c, b, vals(q), [room] * 3, 2)
    assert (kernels.kv8_select(c, b, q, 6, [room, room + 1, 0xFFFFFFFF], 2) == want).all()


@pytest.mark.parametrize("group,kv_heads,kinds,seqs,seq_pages", [(4, 8, [2000, 1990, 40, 2000], 40, 126), (3, 1, [9000, 5, 0, 1], 4, 563)])
def test_attention_writes_over_its_queries(kernels, group, kv_heads, kinds, seqs, seq_pages):
    """out = q: a block writes a row when every slice of its sequence has its queries."""
    from x0ne_core import Arena, Kv8
    from x0ne_core.arena import Class
    rng = np.random.default_rng(group)
    c, of = pooled(rng, kv_heads, kinds, seqs, seq_pages)
    q_heads, lens = group * kv_heads, np.array(kinds, np.uint32)[of]
    q = random_q(rng, 4, q_heads)
    want = kernels.kv8_attention(c, q[of], q_heads, lens, scale=0.088)
    g, a = kernels.gpu, Arena()
    size = g.kv8_work_bytes(Kv8(0, 0, 0, c.pool, kv_heads, seqs, seq_pages), q_heads)
    arrays = {"codes": c.codes, "scales": c.scales, "table": c.table, "q": q[of], "lens": lens, "work": np.zeros(size, np.uint8)}
    s = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()}
    a.freeze(g)
    at = {k: a.ptr(v) for k, v in s.items()}
    for k, v in arrays.items():
        a.write(s[k], 0, np.ascontiguousarray(v))
    kv = Kv8(at["codes"], at["scales"], at["table"], c.pool, kv_heads, seqs, seq_pages)
    for _ in range(3):
        a.write(s["q"], 0, np.ascontiguousarray(q[of]))
        g.kv8_attention(kv, at["q"], q_heads, at["lens"], at["q"], 0.088, at["work"], size)
        g.sync()
        assert (a.read_array(s["q"], 0, want.size, np.uint16).reshape(want.shape) == want).all()
    check_attention(kinds_only(c, 4), q, q_heads, kinds, want[:4], scale=0.088)


def test_sequences_that_share_a_prefix(kernels):
    """Three sequences over the pages of one prompt, each with a page of its own behind them: written into, read back,
    attended and selected from as if the prefix were its own."""
    rng = np.random.default_rng(31)
    kvh, q_heads, prefix, seq_pages = 2, 8, 5, 7
    c = R.fill(rng, kvh, [prefix * PAGE], prefix, spare=9)
    free = [p for p in range(c.pool) if p not in set(c.table[0])]
    table = np.stack([np.concatenate([c.table[0], free[2 * s:2 * s + 2]]) for s in range(3)]).astype(np.uint32)
    c = type(c)(c.codes, c.scales, table)
    counts = [16, 3, 17]
    row_seq = [s for s, n in enumerate(counts) for _ in range(n)]
    row_pos = [prefix * PAGE + i for n in counts for i in range(n)]
    _, c, _ = check_write(kernels, rng, q_heads, kvh, random_qkv(rng, len(row_seq), q_heads, kvh), row_seq, row_pos, seq_pages, 3, cache=c)
    lens = [prefix * PAGE + n for n in counts]
    q = random_q(rng, 3, q_heads)
    check_attention(c, q, q_heads, lens, kernels.kv8_attention(c, q, q_heads, lens))
    b = R.all_bounds(c)
    assert (kernels.kv8_select(c, b, q, q_heads, lens, 3) == R.select(c, b, vals(q), lens, 3)).all()
    out_table = np.arange(3 * seq_pages, dtype=np.uint32).reshape(3, seq_pages)
    check_read(kernels, c, lens, out_table, *kernels.kv8_read(c, lens, out_table, 3 * seq_pages))
