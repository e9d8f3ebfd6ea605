"""The 8-bit paged K/V cache (x0ne_gpu_kv8_*) against its plain 64-bit form (kv8_reference.py): the write bit for
bit, the read-back bit for bit, attention within a derived tolerance, the selected pages exactly."""
import numpy as np
import pytest

import kv8_reference as R
from kv8_reference import HEAD, NONE, PAGE, bits, vals

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-6


# -- write --

def norm_weights(rng):
    return bits(1.0 + 0.2 * rng.standard_normal(HEAD)), bits(1.0 + 0.2 * rng.standard_normal(HEAD))


def check_write(kernels, rng, q_heads, kv_heads, qkv, row_seq, row_pos, seq_pages, seqs, positions=None, table=None,
                with_bounds=True, cache=None):
    """Writes the rows into a garbage cache and compares every byte of it, of q_out and of the bounds."""
    positions = positions or seq_pages * PAGE
    c = cache or R.empty(seqs * seq_pages + 2, kv_heads, seqs, seq_pages, rng)
    if table is not None:
        c.table[...] = table
    qn, kn = norm_weights(rng)
    before = rng.integers(0, 1 << 16, (c.pool, kv_heads, 2, HEAD)).astype(np.uint16) if with_bounds else None
    q, got, bounds = kernels.kv8_write(c, qkv, q_heads, qn, kn, THETA, EPS, positions, row_seq, row_pos, before)
    want_q = np.full(q.shape, kernels.SENTINEL, np.uint16)
    want = type(c)(c.codes.copy(), c.scales.copy(), c.table)
    x = vals(qkv).reshape(len(row_seq), q_heads + 2 * kv_heads, HEAD)
    done = set()
    for r, (s, p) in enumerate(zip(row_seq, row_pos)):
        if s >= seqs or p >= positions or p // PAGE >= seq_pages:
            continue
        want_q[r] = R.rotated(x[r, :q_heads], vals(qn), p, THETA, EPS)
        k = vals(R.rotated(x[r, q_heads:q_heads + kv_heads], vals(kn), p, THETA, EPS))
        R.put(want, s, p, k, x[r, q_heads + kv_heads:])
        if p % PAGE == PAGE - 1 and want.table[s, p // PAGE] < want.pool:
            done.add(int(want.table[s, p // PAGE]))
    nan = np.isnan(vals(want_q))  # a NaN's payload is not stated
    assert ((q == want_q) | (nan & np.isnan(vals(q)))).all(), f"{int((q != want_q).sum())} of q differ"
    assert (got.codes == want.codes).all(), f"{int((got.codes != want.codes).sum())} codes differ"
    assert (got.scales == want.scales).all(), f"{int((got.scales != want.scales).sum())} scale bytes differ"
    if with_bounds:
        for page in range(c.pool):
            w = R.bounds_of(want, page) if page in done else before[page]
            nan = np.isnan(vals(w)) & np.isnan(vals(bounds[page])) if page in done else False
            assert ((bounds[page] == w) | nan).all(), f"bounds of page {page}"
    return q, got, bounds


def random_qkv(rng, rows, q_heads, kv_heads, scale=2.0):
    return bits(scale * rng.standard_normal((rows, (q_heads + 2 * kv_heads) * HEAD))).reshape(rows, -1)


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (16, 8), (32, 8), (64, 8), (3, 3), (14, 2), (5, 1), (20, 4)])
def test_write_of_prompts_and_single_rows(kernels, q_heads, kv_heads):
    """Three sequences' runs (from a page's middle, over two page ends, one row alone) and rows of padding."""
    rng = np.random.default_rng(q_heads * 100 + kv_heads)
    row_seq = [0] * 21 + [2] * 5 + [NONE, 3] + [1]
    row_pos = list(range(27, 48)) + list(range(0, 5)) + [7, 8] + [47]
    check_write(kernels, rng, q_heads, kv_heads, random_qkv(rng, len(row_seq), q_heads, kv_heads), row_seq, row_pos, 4, 3)


@pytest.mark.parametrize("rows,first", [(1, 0), (15, 0), (16, 0), (16, 1), (17, 15), (48, 16), (100, 5), (256, 0)])
def test_write_of_one_prompt(kernels, rows, first):
    rng = np.random.default_rng(rows + first)
    check_write(kernels, rng, 4, 2, random_qkv(rng, rows, 4, 2), [0] * rows, list(range(first, first + rows)), 20, 1)


def test_write_of_whole_pages_of_several_sequences_in_any_order(kernels):
    """Runs of 16 rows that fill pages, rows of one page in falling order (which bounds do not take), and a row at the
    end of another's tile."""
    rng = np.random.default_rng(5)
    row_seq = [1] * 16 + [0] * 16 + [2] * 15 + [0]
    row_pos = list(range(32, 48)) + list(range(31, 15, -1)) + list(range(0, 15)) + [15]
    check_write(kernels, rng, 8, 4, random_qkv(rng, len(row_seq), 8, 4), row_seq, row_pos, 3, 3, with_bounds=False)
    row_pos[16:32] = range(16, 32)
    check_write(kernels, rng, 8, 4, random_qkv(rng, len(row_seq), 8, 4), row_seq, row_pos, 3, 3)


@pytest.mark.parametrize("heads", [(2, 2), (16, 8), (40, 8), (9, 9)])
def test_bounds_of_pages_filled_over_several_calls(kernels, heads):
    """Pages begun by an earlier call and ended by runs that start inside them, over two blocks' rows or one, by single
    rows of a batch, by a run from another block's tile; poison in an old key and in a new one."""
    rng = np.random.default_rng(heads[0])
    seqs, seq_pages = 12, 5
    c = R.fill(rng, heads[1], [5, 12, 15, 31, 14, 15, 47, 0, 79, 63, 30, 1], seq_pages)
    c.codes[c.table[3, 1], 0, 7 * HEAD + 9] = 0x7F
    c.codes[c.table[3, 1], 0, 15 * HEAD:16 * HEAD] = 0x7F
    runs = [(0, 5, 40), (1, 12, 4), (2, 15, 1), (3, 31, 1), (4, 14, 2), (5, 15, 18), (6, 47, 1), (7, 0, 16), (8, 79, 1),
            (9, 63, 1), (10, 30, 30), (11, 1, 15)]
    row_seq = [s for s, _, n in runs for _ in range(n)]
    row_pos = [p + i for _, p, n in runs for i in range(n)]
    qkv = random_qkv(rng, len(row_seq), *heads)
    qkv.reshape(len(row_seq), -1, HEAD)[43, heads[0], 100] = 0x7FC0  # a key of sequence 1's page
    check_write(kernels, rng, *heads, qkv, row_seq, row_pos, seq_pages, seqs, cache=c)


@pytest.mark.parametrize("kv_heads", [1, 6, 7])
def test_bounds_of_a_launch_of_many_blocks(kernels, kv_heads):
    """Heads enough that a block takes four of them: a prompt that starts inside a page (each page's rows in two
    blocks, the first with slots of an earlier call), then one whole page, then single rows that end pages."""
    rng = np.random.default_rng(kv_heads)
    q_heads = 2048 // kv_heads * kv_heads
    c = R.fill(rng, kv_heads, [5, 16, 31, 47], 5)
    row_seq = [0] * 43 + [1] * 5 + [1] * 16 + [2, 3]
    row_pos = list(range(5, 48)) + list(range(16, 21)) + list(range(32, 48)) + [31, 47]
    check_write(kernels, rng, q_heads, kv_heads, random_qkv(rng, len(row_seq), q_heads, kv_heads), row_seq, row_pos, 5, 4, cache=c)


def test_rows_past_the_table_or_the_pool_are_left_alone(kernels):
    """Padding of every kind: no such sequence, past the sequence's pages, past the rope table, a page outside the
    pool (its q is written); the bounds of a page outside the pool are not."""
    rng = np.random.default_rng(6)
    table = np.array([[3, 4], [0xFFFFFFFF, 1], [6, 0]], np.uint32)
    c = R.empty(6, 2, 3, 2)
    row_seq = [0, 0, 1, 1, 1, 2, 2, 2, 9, NONE]
    row_pos = [31, 32, 15, 3, 16, 15, 16, 0xFFFFFFFF, 0, 1]
    check_write(kernels, rng, 4, 2, random_qkv(rng, 10, 4, 2), row_seq, row_pos, 2, 3, positions=64, table=table, cache=c)
    c = R.empty(6, 2, 3, 2)
    check_write(kernels, rng, 4, 2, random_qkv(rng, 10, 4, 2), row_seq, row_pos, 2, 3, positions=16, cache=c)


def test_every_bf16_value_is_held_as_its_nearest_code(kernels):
    """All 2^16 patterns as values, 128 per row, alone (their own scale) and beside 1, 300 and 3e38 (given scales):
    rows with infinities and NaN, zeros, denormals, the largest values."""
    patterns = np.arange(1 << 16, dtype=np.uint32).astype(np.uint16)
    rows = [patterns.reshape(-1, HEAD)]
    for x in (1.0, 300.0, 3e38):
        sample = patterns[::64].reshape(-1, HEAD).copy()
        sample[:, 0] = bits([x])[0]
        rows.append(sample)
    v = np.concatenate(rows)
    n = v.shape[0]
    rng = np.random.default_rng(7)
    qkv = random_qkv(rng, n, 1, 1)
    qkv[:, 2 * HEAD:] = v
    check_write(kernels, rng, 1, 1, qkv, [0] * n, list(range(n)), -(-n // PAGE), 1)


@pytest.mark.parametrize("special", [0.0, -0.0, 1e-38, 1e-30, 3e38, np.inf, -np.inf, np.nan])
def test_keys_of_special_values(kernels, special):
    """A head of q and of k all special, one with a single such value: norms of zero rows, of rows whose squares
    pass f32, rows that are not finite (poison: NaN codes, NaN bounds)."""
    rng = np.random.default_rng(8)
    qkv = random_qkv(rng, 32, 2, 2).reshape(32, 6, HEAD)
    qkv[3, 0] = qkv[4, 2] = qkv[9, 3] = bits(np.full(HEAD, special))
    qkv[5, 1, 17] = qkv[6, 2, 99] = bits([special])[0]
    with np.errstate(invalid="ignore", over="ignore"):
        check_write(kernels, rng, 2, 2, qkv.reshape(32, -1), [0] * 32, list(range(32)), 2, 1)


def test_the_write_is_the_bf16_write_quantised(kernels):
    """q_out and the codes against the bf16 cache's own kernel on the same row."""
    from x0ne_core.ops import CacheAt, Heads
    rng = np.random.default_rng(9)
    for q_heads, kv_heads, pos in [(16, 8, 0), (32, 8, 4097), (64, 8, 333)]:
        qkv = random_qkv(rng, 1, q_heads, kv_heads)
        qn, kn = norm_weights(rng)
        bf = kernels.qk_norm_rope_kv_write(qkv[0], qn, kn, Heads(q_heads, kv_heads), THETA, EPS,
                                           CacheAt(1, pos + 1, 0, pos), table=True)
        c = R.empty(pos // PAGE + 1, kv_heads, 1, pos // PAGE + 1)
        q, got, _ = kernels.kv8_write(c, qkv, q_heads, qn, kn, THETA, EPS, pos + 1, [0], [pos])
        assert (q.reshape(-1) == bf.q).all()
        want = R.empty(c.pool, kv_heads, 1, c.table.shape[1])
        R.put(want, 0, pos, vals(bf.k_row).reshape(kv_heads, HEAD), vals(bf.v_row).reshape(kv_heads, HEAD))
        assert (got.codes == want.codes).all() and (got.scales == want.scales).all()


# -- read --

@pytest.mark.parametrize("kv_heads,lens", [(1, [1]), (8, [333]), (2, [0, 16, 17, 15, 48]), (3, [64, 1, 0]), (8, [0])])
def test_read_back(kernels, kv_heads, lens):
    """Exact bf16 values below the length, zeros behind it in its last page, everything else left alone."""
    rng = np.random.default_rng(sum(lens) + kv_heads)
    seq_pages = max(lens) // PAGE + 2
    c = R.fill(rng, kv_heads, lens, seq_pages)
    out_pool = len(lens) * seq_pages + 1
    out_table = rng.permutation(out_pool)[:len(lens) * seq_pages].reshape(len(lens), seq_pages).astype(np.uint32)
    k, v = kernels.kv8_read(c, lens, out_table, out_pool)
    check_read(kernels, c, lens, out_table, k, v)


def test_read_under_a_table_far_wider_than_the_sequences(kernels):
    rng = np.random.default_rng(12)
    lens = [0, 1000, 17]
    c = R.fill(rng, 2, lens, 64)
    out_table = np.full((3, 9000), NONE, np.uint32)
    out_table[:, :64] = rng.permutation(200)[:192].reshape(3, 64)
    k, v = kernels.kv8_read(widened(c, 9000), lens, out_table, 200)
    check_read(kernels, c, lens, out_table, k, v)


def test_read_of_more_records_than_wavefronts(kernels):
    """100000 pages of 3 kv heads: a wavefront takes several. The pages are five in turn, most go nowhere."""
    rng = np.random.default_rng(25)
    pages, kvh = 100000, 3
    c = R.fill(rng, kvh, [80], 5, spare=0)
    c = type(c)(c.codes, c.scales, np.resize(c.table, (1, pages)))
    at = [0, 1, 43690, 43691, 87380, 87381, 87382, 99998, 99999]
    out_table = np.full((1, pages), NONE, np.uint32)
    out_table[0, at] = np.arange(len(at))
    lens = [pages * PAGE - 5]
    k, v = kernels.kv8_read(c, lens, out_table, len(at))
    for i, p in enumerate(at):
        want_k, want_v = R.page_values(c, int(c.table[0, p]))
        if p == pages - 1:
            want_k[:, 11:], want_v[:, 11:] = 0, 0
        assert (vals(k[i]).reshape(kvh, PAGE, HEAD) == want_k).all() and (vals(v[i]).reshape(kvh, HEAD, PAGE) == want_v.transpose(0, 2, 1)).all(), p


def check_read(kernels, c, lens, out_table, k, v):
    want_k, want_v = np.full(k.shape, kernels.SENTINEL, np.uint16), np.full(v.shape, kernels.SENTINEL, np.uint16)
    for s, n in enumerate(lens):
        n = min(n, c.table.shape[1] * PAGE)
        for p in range(-(-n // PAGE)):
            to, at = int(out_table[s, p]), int(c.table[s, p])
            if to >= k.shape[0]:
                continue
            kk, vv = np.zeros((2, c.kv_heads, PAGE, HEAD))
            if at < c.pool:
                kk, vv = (x.copy() for x in R.page_values(c, at))
                kk[:, n - p * PAGE:], vv[:, n - p * PAGE:] = 0.0, 0.0
            want_k[to], want_v[to] = bits(kk).reshape(kk.shape), bits(vv).reshape(vv.shape).transpose(0, 2, 1)
    for got, want in ((k, want_k), (v, want_v)):
        nan = np.isnan(vals(want)) & np.isnan(vals(got))
        assert ((got == want) | nan).all(), f"{int((got != want).sum())} values differ"


def test_read_of_every_code_under_every_scale_that_is_written(kernels):
    """All 256 codes under the scale bytes 10 to 247; a length past the pages; missing and unwritable pages."""
    rng = np.random.default_rng(11)
    c = R.fill(rng, 2, [16 * 15, 16 * 15], 15)
    c.codes[...] = rng.integers(0, 256, c.codes.shape)
    c.codes.reshape(-1)[:256] = np.arange(256)
    c.scales[...] = rng.integers(10, 248, c.scales.shape)
    c.scales.reshape(-1)[:238] = np.arange(10, 248)
    c.table[0, 3], c.table[1, 7] = c.pool, 0xFFFFFFFF
    out_table = np.arange(30, dtype=np.uint32).reshape(2, 15)
    out_table[1, 2], out_table[0, 5] = 30, 0xFFFFFFFF
    lens = [16 * 15 - 3, 10 ** 6]
    k, v = kernels.kv8_read(c, lens, out_table, 30)
    check_read(kernels, c, lens, out_table, k, v)


# -- attention --

def tolerance(keys, vmax, reach):
    """How far an output may be from its 64-bit value, beside the rounding to bf16 (half a step: 2^-8 of it). A score
    is a sum of 128 products in f32 in any order, off by at most 130 2^-24 of `reach` (the largest sum |q k| times
    the scale's magnitude), and its weight by e to twice that with the maximum's; a weight enters the value sums as two bf16
    parts (2^-17 of it) or in f32; sums of `keys` terms and joins in f32 add (keys + 64) 2^-24, the exponential
    and the division a few 2^-23 each. Numerator and denominator both: twice."""
    return 2 * vmax * (4 * 130 * 2.0 ** -24 * reach + 2.0 ** -16 + (keys + 64) * 2.0 ** -24 + 2.0 ** -20)


def check_attention(c, q, q_heads, lens, out, page_list=None, scale=None):
    from x0ne_core.ops import attn_scale
    scale = attn_scale(HEAD) if scale is None else float(np.float32(scale))
    group, worst = q_heads // c.kv_heads, 0.0
    qv, got = vals(q).reshape(len(lens), c.kv_heads, group, HEAD), vals(out).reshape(len(lens), c.kv_heads, group, HEAD)
    for s, n in enumerate(lens):
        limit = -(-min(int(n), c.table.shape[1] * PAGE) // PAGE)
        for h in range(c.kv_heads):
            pages = None
            if page_list is not None:
                pages = [int(p) for p in page_list[s, h, :min(page_list.shape[-1], limit)] if p < limit]
            k, v = R.sequence(c, s, int(n), pages)
            want, reach = R.attention(qv[s, h], k[h], v[h], scale)
            nan = np.isnan(want)
            assert (np.isnan(got[s, h]) == nan).all(), f"sequence {s}, kv head {h}: NaN at other places"
            if nan.all():
                continue
            tol = tolerance(k.shape[1], float(np.nanmax(np.abs(v[h]))) if k.shape[1] else 0.0, reach) + 2.0 ** -8 * np.abs(want)
            off = np.abs(got[s, h] - want)[~nan]
            with np.errstate(invalid="ignore", divide="ignore"):
                worst = max(worst, float(np.nanmax(np.where(off == 0, 0.0, off / np.broadcast_to(tol, want.shape)[~nan]))))
            assert (off <= np.broadcast_to(tol, want.shape)[~nan]).all(), f"sequence {s} of {n} keys, kv head {h}: {off.max()} off"
    print(f"MEASURE kv8 attention {q_heads}/{c.kv_heads} {list(lens)[:6]}: worst {worst:.3f} of the tolerance")


def random_q(rng, seqs, q_heads, scale=1.5):
    return bits(scale * rng.standard_normal((seqs, q_heads, HEAD))).reshape(seqs, q_heads, HEAD)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 12, 16])
@pytest.mark.parametrize("kv_heads", [1, 3, 8])
def test_attention_of_every_group(kernels, group, kv_heads):
    rng = np.random.default_rng(group * 10 + kv_heads)
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 130, 257]
    c = R.fill(rng, kv_heads, lens, 17)
    q = random_q(rng, len(lens), group * kv_heads)
    out = kernels.kv8_attention(c, q, group * kv_heads, lens)
    assert (out[0] == 0).all()
    check_attention(c, q, group * kv_heads, lens, out)
    again = kernels.kv8_attention(c, q, group * kv_heads, lens, calls=3)
    assert (again == out).all(), "a repeated call over the same workspace"


@pytest.mark.parametrize("seqs,longest", [(1, 300), (1, 1025), (1, 4097), (1, 20000), (2, 9000), (7, 2500), (40, 700)])
def test_attention_of_ragged_batches(kernels, seqs, longest):
    """Lengths spread over the range, more pages in the table than any sequence uses."""
    rng = np.random.default_rng(seqs + longest)
    lens = [longest] + [int(x) for x in rng.integers(0, longest + 1, seqs - 1)]
    c = R.fill(rng, 2, lens, longest // PAGE + 9, drift=2.0)
    q = random_q(rng, seqs, 8)
    out = kernels.kv8_attention(c, q, 8, lens)
    check_attention(c, q, 8, lens, out)
    assert (kernels.kv8_attention(c, q, 8, lens, calls=2) == out).all()


def widened(c, seq_pages):
    """The same cache under a table of seq_pages entries, those past the sequences' naming no page."""
    table = np.full((c.table.shape[0], seq_pages), NONE, np.uint32)
    table[:, :c.table.shape[1]] = c.table
    return type(c)(c.codes, c.scales, table)


@pytest.mark.parametrize("q_heads,kv_heads,lens", [(8, 8, [2000]), (24, 8, [0, 700, 33, 1, 512, 4000]), (5, 1, [9000]),
                                                   (16, 1, [16, 3333, 0]), (14, 2, [1000] * 9 + [17]), (32, 4, [6001, 5, 90])])
def test_attention_under_tables_far_wider_than_the_sequences(kernels, q_heads, kv_heads, lens):
    """Tables that hold millions of positions: blocks of 8 wavefronts and the cuts that go with them, at every group
    that joins in another number of parts; lists of pages under the same tables."""
    rng = np.random.default_rng(q_heads)
    c = R.fill(rng, kv_heads, lens, max(lens) // PAGE + 1)
    q = random_q(rng, len(lens), q_heads)
    for width in (c.table.shape[1], 3000, 20000, 200000):
        wide = widened(c, width)
        out = kernels.kv8_attention(wide, q, q_heads, lens, calls=2)
        check_attention(c, q, q_heads, lens, out)
    pages = np.full((len(lens), kv_heads, 4096), NONE, np.uint32)
    for s, n in enumerate(lens):
        for h in range(kv_heads):
            pick = np.sort(rng.permutation(-(-n // PAGE))[:200])
            pages[s, h, :len(pick)] = pick
    out = kernels.kv8_attention(widened(c, 20000), q, q_heads, lens, page_list=pages)
    check_attention(c, q, q_heads, lens, out, page_list=pages)


@pytest.mark.parametrize("seqs,kv_heads", [(70, 8), (130, 2), (65, 1), (300, 1)])
def test_attention_of_more_than_64_sequences(kernels, seqs, kv_heads):
    """Batches in several parts of 64, sequences of all lengths, empty ones among them, each block with several."""
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(0, 200, seqs)]
    lens[::7] = [0] * len(lens[::7])
    lens[-1], lens[63], lens[64] = 333, 1, 600
    c = R.fill(rng, kv_heads, lens, 40)
    q = random_q(rng, seqs, 3 * kv_heads)
    out = kernels.kv8_attention(c, q, 3 * kv_heads, lens, calls=2)
    check_attention(c, q, 3 * kv_heads, lens, out)


def test_a_sequence_has_its_bits_in_any_batch(kernels):
    """The same sequence beside others of any lengths, at another place of the batch: the same bits."""
    rng = np.random.default_rng(21)
    lens = [3000, 17, 2000, 900, 0, 4000, 64, 3000]
    c = R.fill(rng, 2, lens, 260)
    q = random_q(rng, 8, 8)
    first = kernels.kv8_attention(c, q, 8, lens)
    order = rng.permutation(8)
    moved = type(c)(c.codes, c.scales, c.table[order])
    again = kernels.kv8_attention(moved, q[order], 8, [lens[i] for i in order])
    assert (again == first[order]).all()
    alone = list(lens)
    for i in range(8):
        if i not in (0, 3):
            alone[i] = 0
    other = kernels.kv8_attention(c, q, 8, alone)
    assert (other[[0, 3]] == first[[0, 3]]).all()


def test_attention_of_sharp_and_flat_scores(kernels):
    """Scores far apart (one key takes all), a scale of 0 (the mean of the values), and a negative scale."""
    rng = np.random.default_rng(13)
    lens = [500, 1100]
    c = R.fill(rng, 2, lens, 80)
    for s, scale in ((60.0, None), (1.5, 0.0), (1.5, -0.3)):
        q = random_q(rng, 2, 6, s)
        check_attention(c, q, 6, lens, kernels.kv8_attention(c, q, 6, lens, scale=scale), scale=scale)


def test_attention_passes_over_missing_pages_and_clamps_lengths(kernels):
    """Entries outside the pool hold no keys: some, a whole slice of them, all of a sequence's; a length past the
    table's pages reads what they hold."""
    rng = np.random.default_rng(14)
    lens = [400, 700, 90, 1700, 5 * 10 ** 8]
    c = R.fill(rng, 2, lens, 110)
    c.table[0, 3], c.table[0, 24], c.table[1, :40], c.table[2, :] = c.pool, 0xFFFFFFFF, c.pool + 7, 0xFFFFFFF0
    c.table[3, 5:100] = c.pool
    q = random_q(rng, 5, 8)
    out = kernels.kv8_attention(c, q, 8, lens)
    assert (out[2] == 0).all()
    check_attention(c, q, 8, lens, out)


def test_attention_keeps_poison_to_its_own(kernels):
    """A NaN in a key: every head of that kv head; in a value: that dim; other sequences and heads as without."""
    rng = np.random.default_rng(15)
    lens = [300, 300, 300]
    c = R.fill(rng, 2, lens, 20)
    q = random_q(rng, 3, 8)
    clean = kernels.kv8_attention(c, q, 8, lens)
    c.codes[c.table[1, 7], 0, 5 * HEAD + 3] = 0xFF
    c.codes[c.table[2, 18], 1, 2048 + 77 * PAGE + 2] = 0x7F
    out = kernels.kv8_attention(c, q, 8, lens)
    check_attention(c, q, 8, lens, out)
    same = np.ones_like(out, bool)
    same[1, :4] = False
    same[2, 4:, 77] = False
    assert (out[same] == clean[same]).all()
    assert np.isnan(vals(out)[1, :4]).all() and np.isnan(vals(out)[2, 4:, 77]).all()


@pytest.mark.parametrize("kv_heads,lens", [(2, [5, 0, 40, 700]), (1, [9000]), (8, [300] * 20)])
def test_attention_of_queries_that_hold_an_infinity(kernels, kv_heads, lens):
    """Keys whose dim 7 is positive and queries with -inf or +inf there: every score -inf or +inf, whose softmax is NaN;
    the other heads and sequences have the bits they have without."""
    rng = np.random.default_rng(23)
    c = R.fill(rng, kv_heads, lens, -(-max(lens) // PAGE))
    row = c.codes[:, :, :2048].reshape(c.pool, kv_heads, PAGE, HEAD)
    row[..., 7] = np.maximum(row[..., 7] & 0x7F, 1)
    clean = random_q(rng, len(lens), 4 * kv_heads)
    q, bad = clean.copy(), np.zeros(clean.shape[:2], bool)
    for s, h, x in [(0, 0, 0xFF80), (-1, -1, 0xFF80), (-1, 1, 0x7F80)]:
        q[s, h, 7] = x
        bad[s, h] = True
    out = kernels.kv8_attention(c, q, 4 * kv_heads, lens)
    check_attention(c, q, 4 * kv_heads, lens, out)
    assert np.isnan(vals(out)[bad]).all() and (out[~bad] == kernels.kv8_attention(c, clean, 4 * kv_heads, lens)[~bad]).all()


@pytest.mark.parametrize("budget", [1, 2, 5, 16, 70])
def test_attention_over_a_page_list(kernels, budget):
    """Lists of chosen pages (with and without the last), shorter than the budget, entries of none among them."""
    rng = np.random.default_rng(budget)
    lens = [1000, 37, 0, 16, 640]
    c = R.fill(rng, 2, lens, 66)
    c.table[4, 11] = c.pool
    pages = np.full((5, 2, budget), NONE, np.uint32)
    for s, n in enumerate(lens):
        for h in range(2):
            total = -(-n // PAGE)
            pick = np.sort(rng.permutation(total)[:budget - (budget > 4 and h)])
            pages[s, h, :len(pick)] = pick
    if budget > 4:
        pages[0, 0, 2] = 63  # the page behind the last one
    q = random_q(rng, 5, 8)
    out = kernels.kv8_attention(c, q, 8, lens, page_list=pages)
    check_attention(c, q, 8, lens, out, page_list=pages)


def test_attention_and_write_in_a_pool_past_4_gib(kernels):
    """Pages whose records lie past 2^32 bytes: what is written there is read, by every call."""
    from x0ne_core import Arena, Kv8
    from x0ne_core.arena import Class
    rng = np.random.default_rng(16)
    pool, kvh, seq_pages = (1 << 20) + 4096 + 40, 1, 40
    n = 16 * seq_pages - 5
    table = (pool - 1 - rng.permutation(seq_pages)).astype(np.uint32)[None]
    small = R.fill(rng, kvh, [n], seq_pages, spare=0)
    bounds = R.all_bounds(small)
    g = kernels.gpu
    arrays = {"table": table, "lens": np.array([n], np.uint32), "q": random_q(rng, 1, 4), "list": np.zeros(8, np.uint32),
              "out_table": np.arange(seq_pages, dtype=np.uint32)}
    a = Arena()
    s = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()}
    size = g.kv8_work_bytes(Kv8(16, 16, 16, pool, kvh, 1, seq_pages), 4)
    for name, length in {"codes": pool * 4096, "scales": pool * 32, "bounds": pool * 512, "work": size, "out": 1024,
                         "k": seq_pages * 4096, "v": seq_pages * 4096}.items():
        s[name] = a.alloc(name, length, Class.CLIENT_DATA)
    a.freeze(g)
    for k, v in arrays.items():
        a.write(s[k], 0, v)
    a.write(s["work"], 0, np.zeros(size, np.uint8))
    for p in range(seq_pages):
        at, to = int(small.table[0, p]), int(table[0, p])
        a.write(s["codes"], to * 4096, small.codes[at])
        a.write(s["scales"], to * 32, small.scales[at])
        a.write(s["bounds"], to * 512, bounds[at])
    kv = Kv8(a.ptr(s["codes"]), a.ptr(s["scales"]), a.ptr(s["table"]), pool, kvh, 1, seq_pages)
    g.kv8_select(kv, a.ptr(s["bounds"]), a.ptr(s["q"]), 4, a.ptr(s["lens"]), 8, a.ptr(s["list"]), a.ptr(s["work"]), size)
    pages = a.read_array(s["list"], 0, 8, np.uint32).reshape(1, 1, 8)
    assert (pages == R.select(small, bounds, vals(arrays["q"]), [n], 8)).all()
    for extra in ({}, {"page_list": a.ptr(s["list"]), "budget": 8}):
        g.kv8_attention(kv, a.ptr(s["q"]), 4, a.ptr(s["lens"]), a.ptr(s["out"]), 0.088, a.ptr(s["work"]), size, **extra)
        out = a.read_array(s["out"], 0, 512, np.uint16).reshape(1, 4, HEAD)
        check_attention(small, arrays["q"], 4, [n], out, page_list=pages if extra else None, scale=0.088)
    g.kv8_read(kv, a.ptr(s["lens"]), a.ptr(s["k"]), a.ptr(s["v"]), a.ptr(s["out_table"]), seq_pages)
    k = a.read_array(s["k"], 0, seq_pages * 2048, np.uint16).reshape(seq_pages, 1, PAGE, HEAD)
    v = a.read_array(s["v"], 0, seq_pages * 2048, np.uint16).reshape(seq_pages, 1, HEAD, PAGE)
    check_read(kernels, small, [n], arrays["out_table"][None], k, v)


# -- selection --

@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 2), (32, 8), (7, 7), (48, 4), (16, 1)])
@pytest.mark.parametrize("budget", [1, 2, 7, 64, 300])
def test_selected_pages(kernels, q_heads, kv_heads, budget):
    rng = np.random.default_rng(q_heads * budget + kv_heads)
    lens = [0, 1, 16, 17, 16 * budget, 16 * budget + 1, 900, 4001]
    c = R.fill(rng, kv_heads, lens, 304 if budget == 300 else 251, drift=2.0)
    b, q = R.all_bounds(c), random_q(rng, len(lens), q_heads)
    want = R.select(c, b, vals(q), lens, budget)
    got = kernels.kv8_select(c, b, q, q_heads, lens, budget)
    assert (got == want).all()
    assert (kernels.kv8_select(c, b, q, q_heads, lens, budget, calls=3) == want).all()


def test_selection_among_ties_missing_pages_and_nan(kernels):
    """Equal scores go to the lower page (all equal; runs of equal ones; zeros of both signs), missing pages come
    last, pages with NaN bounds first, a query of NaN or infinities still picks within the sequence."""
    rng = np.random.default_rng(17)
    pages = 700
    lens = [pages * PAGE - 3] * 4
    c = R.empty(4 * pages + 1, 2, 4, pages, rng)
    b = bits(rng.standard_normal((c.pool, 2, 2, HEAD))).reshape(c.pool, 2, 2, HEAD)
    b[c.table[0]] = b[0]
    b[c.table[1]] = b[c.table[1]][rng.integers(0, 5, pages)]
    b[c.table[2, 3:300]] = 0
    b[c.table[2, 300:600]] = 0x8000
    b[c.table[3, ::9], 0, 1, 5] = 0x7FC0
    c.table[3, 1::3] = 0xFFFFFFFF
    c.table[0, 4] = c.pool
    q = random_q(rng, 4, 8)
    for budget in (1, 9, 333, 699, 700, 701):
        assert (kernels.kv8_select(c, b, q, 8, lens, budget) == R.select(c, b, vals(q), lens, budget)).all(), budget
    q[0, 0], q[1, 4:, 3] = 0x7FC0, 0x7F80
    got = kernels.kv8_select(c, b, q, 8, lens, 20)
    assert (got == R.select(c, b, vals(q), lens, 20)).all()


@pytest.mark.parametrize("pages,seqs", [(4098, 1), (9001, 2), (257, 3), (258, 3), (65, 2), (66, 2)])
def test_selection_of_any_number_of_pages(kernels, pages, seqs):
    """Pages that one block scores and one more, more than a block's threads hold at once, under tables as wide as they
    and far wider; scores of few values (ties over all of them), of all signs, of both zeros."""
    rng = np.random.default_rng(pages)
    lens = [pages * PAGE - 7] + [(pages - 30 * (s + 1)) * PAGE for s in range(seqs - 1)]
    c = R.empty(pages + 5, 1, seqs, pages // seqs, rng)
    c.table = rng.integers(0, c.pool, (seqs, pages)).astype(np.uint32)
    few = bits(rng.integers(-2, 3, (c.pool, 1, 2, HEAD)) * (rng.random((c.pool, 1, 2, HEAD)) < 0.02)).reshape(-1, 1, 2, HEAD)
    many = bits(rng.standard_normal((c.pool, 1, 2, HEAD))).reshape(-1, 1, 2, HEAD)
    for b in (few, many):
        q = random_q(rng, seqs, 2) if b is many else bits(np.sign(rng.standard_normal((seqs, 2, HEAD)))).reshape(seqs, 2, HEAD)
        for budget in (2, 33, pages - 40):
            want = R.select(c, b, vals(q), lens, budget)
            for width in (pages, 40000):
                assert (kernels.kv8_select(widened(c, width), b, q, 2, lens, budget, calls=2) == want).all(), (budget, width)


@pytest.mark.parametrize("q_heads,kv_heads", [(16, 1), (8, 8), (15, 3)])
def test_selected_pages_under_wide_tables(kernels, q_heads, kv_heads):
    rng = np.random.default_rng(q_heads)
    lens = [0, 1, 300, 1030, 1040, 4112, 6000]
    c = R.fill(rng, kv_heads, lens, 376, drift=2.0)
    b, q = R.all_bounds(c), random_q(rng, len(lens), q_heads)
    for budget in (2, 40):
        assert (kernels.kv8_select(widened(c, 30000), b, q, q_heads, lens, budget) == R.select(c, b, vals(q), lens, budget)).all()


# -- together --

def test_a_conversation_through_the_cache(kernels):
    """Prompts of three sequences written, read back into bf16 pages and attended causally by the bf16 prefill
    kernel; then tokens decoded one by one: written (pages filled, bounds kept), pages selected, attended over all
    pages and over the chosen ones. The step (write, select, both attentions) is a captured graph, replayed with
    eager steps and synchronisations between, each against the plain form."""
    from x0ne_core import Arena, Kv8
    from x0ne_core.arena import Class
    from x0ne_core.gpu import Arg
    from x0ne_core.ops import attn_scale, inv_freq
    rng = np.random.default_rng(18)
    q_heads, kvh, seqs, seq_pages, budget, prompts = 8, 2, 3, 12, 3, [61, 16, 130]
    pool, positions, rows = seqs * seq_pages + 2, seq_pages * PAGE, sum(prompts)
    g, qn, kn = kernels.gpu, *norm_weights(rng)
    want = R.empty(pool, kvh, seqs, seq_pages, rng)
    steps = 20
    line = (q_heads + 2 * kvh) * HEAD
    token_qkv = random_qkv(rng, steps * seqs, q_heads, kvh)
    prompt_qkv = random_qkv(rng, rows, q_heads, kvh)
    row_seq = np.concatenate([[s] * n for s, n in enumerate(prompts)]).astype(np.uint32)
    row_pos = np.concatenate([np.arange(n) for n in prompts]).astype(np.uint32)
    a = Arena()
    plan = {"codes": want.codes.nbytes, "scales": want.scales.nbytes, "bounds": pool * kvh * 512, "table": want.table.nbytes,
            "cs": positions * 1024, "inv": 256, "qn": 256, "kn": 256, "prompt": prompt_qkv.nbytes, "seq": 4 * rows,
            "pos": 4 * rows, "pq": rows * q_heads * 256, "k": pool * kvh * 4096, "v": pool * kvh * 4096, "pos0": 4,
            "prefill": rows * q_heads * 256, "qkv": seqs * line * 2, "tseq": 4 * seqs, "tpos": 4 * seqs, "lens": 4 * seqs,
            "q": seqs * q_heads * 256, "out": seqs * q_heads * 256, "sparse": seqs * q_heads * 256, "list": seqs * kvh * budget * 4}
    plan["work"] = g.kv8_work_bytes(Kv8(16, 16, 16, pool, kvh, seqs, seq_pages), q_heads)
    sl = {k: a.alloc(k, n, Class.CLIENT_DATA) for k, n in plan.items()}
    a.freeze(g)
    a.scrub_client_data()
    at = {k: a.ptr(v) for k, v in sl.items()}
    for k, x in {"codes": want.codes, "scales": want.scales, "table": want.table, "inv": inv_freq(HEAD, THETA), "qn": qn, "kn": kn,
                 "prompt": prompt_qkv, "seq": row_seq, "pos": row_pos, "lens": np.array(prompts, np.uint32),
                 "tseq": np.arange(seqs, dtype=np.uint32)}.items():
        a.write(sl[k], 0, x)
    kernels._rope_table(at["inv"], at["cs"], positions, HEAD)
    kv = Kv8(at["codes"], at["scales"], at["table"], pool, kvh, seqs, seq_pages)
    scale = attn_scale(HEAD)

    def reference_row(x, s, p):
        x = vals(x).reshape(-1, HEAD)
        R.put(want, s, p, vals(R.rotated(x[q_heads:q_heads + kvh], vals(kn), p, THETA, EPS)), x[q_heads + kvh:])
        return R.rotated(x[:q_heads], vals(qn), p, THETA, EPS)

    # prompts
    g.kv8_write(kv, at["prompt"], rows, q_heads, at["qn"], at["kn"], EPS, at["cs"], positions, at["seq"], at["pos"], at["pq"],
                bounds=at["bounds"])
    g.kv8_read(kv, at["lens"], at["k"], at["v"], at["table"], pool)
    first = 0
    for s, n in enumerate(prompts):
        g.launch("x0ne_attention_prefill_g4_bf16", (kvh, -(-n // 32)), 256,
                 [Arg.ptr(at["pq"] + first * q_heads * 256), Arg.ptr(at["k"]), Arg.ptr(at["v"]),
                  Arg.ptr(at["table"] + s * seq_pages * 4), Arg.ptr(at["prefill"] + first * q_heads * 256), Arg.ptr(at["pos0"]),
                  Arg.u32(n), Arg.u32(q_heads), Arg.u32(kvh), Arg.u32(positions), Arg.f32(scale)])
        first += n
    g.sync()
    q_ref = np.stack([reference_row(prompt_qkv[r], int(row_seq[r]), int(row_pos[r])) for r in range(rows)])
    assert (a.read_array(sl["pq"], 0, rows * q_heads * HEAD, np.uint16).reshape(q_ref.shape) == q_ref).all()
    got = vals(a.read_array(sl["prefill"], 0, rows * q_heads * HEAD, np.uint16)).reshape(rows, kvh, 4, HEAD)
    for r in range(rows):
        k, v = R.sequence(want, int(row_seq[r]), int(row_pos[r]) + 1)
        for h in range(kvh):
            ref, _ = R.attention(vals(q_ref[r]).reshape(kvh, 4, HEAD)[h], k[h], v[h], scale)
            assert (np.abs(got[r, h] - ref) <= np.abs(v[h]).max() / 128 + 2.0 ** -8 * np.abs(ref)).all(), r

    # tokens
    def step():
        g.kv8_write(kv, at["qkv"], seqs, q_heads, at["qn"], at["kn"], EPS, at["cs"], positions, at["tseq"], at["tpos"], at["q"],
                    bounds=at["bounds"])
        g.kv8_select(kv, at["bounds"], at["q"], q_heads, at["lens"], budget, at["list"], at["work"], plan["work"])
        g.kv8_attention(kv, at["q"], q_heads, at["lens"], at["out"], scale, at["work"], plan["work"])
        g.kv8_attention(kv, at["q"], q_heads, at["lens"], at["sparse"], scale, at["work"], plan["work"], page_list=at["list"],
                        budget=budget)

    graph = g.capture(step)
    lens = list(prompts)
    for t in range(steps):
        x = token_qkv[t * seqs:(t + 1) * seqs]
        pos = list(lens)
        lens = [n + 1 for n in lens]
        for k, v in {"qkv": x, "tpos": np.array(pos, np.uint32), "lens": np.array(lens, np.uint32)}.items():
            a.write(sl[k], 0, v)
        if t % 5 == 2:
            step()
        else:
            g.launch_graph(graph)
        g.sync()
        q = np.stack([reference_row(x[s], s, pos[s]) for s in range(seqs)])
        assert (a.read_array(sl["q"], 0, q.size, np.uint16).reshape(q.shape) == q).all()
        assert (a.read_array(sl["codes"], 0, want.codes.size, np.uint8).reshape(want.codes.shape) == want.codes).all()
        check_attention(want, q, q_heads, lens, a.read_array(sl["out"], 0, q.size, np.uint16))
        pages = a.read_array(sl["list"], 0, seqs * kvh * budget, np.uint32).reshape(seqs, kvh, budget)
        assert (pages == R.select(want, R.all_bounds(want), vals(q), lens, budget)).all()
        check_attention(want, q, q_heads, lens, a.read_array(sl["sparse"], 0, q.size, np.uint16), page_list=pages)


def test_two_calls_of_a_batch_on_one_workspace_do_not_meet(kernels):
    """Batches of two shapes in turn over one workspace, as two graphs of a program replay: each the bits it has
    alone."""
    from x0ne_core import Arena, Kv8
    from x0ne_core.arena import Class
    rng = np.random.default_rng(19)
    g, a, calls, keep = kernels.gpu, Arena(), [], []
    shapes = [(2, 8, [5000, 800]), (1, 4, [3000]), (4, 12, [100, 0, 2100, 17])]
    size = 0
    for kvh, q_heads, lens in shapes:
        c = R.fill(rng, kvh, lens, 320)
        q = random_q(rng, len(lens), q_heads)
        kv = Kv8(16, 16, 16, c.pool, kvh, *c.table.shape)
        size = max(size, g.kv8_work_bytes(kv, q_heads))
        arrays = {"codes": c.codes, "scales": c.scales, "table": c.table, "q": q, "lens": np.array(lens, np.uint32)}
        keep.append((c, q, q_heads, lens, {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()}, arrays,
                     a.alloc("out", q.nbytes, Class.CLIENT_DATA)))
    work = a.alloc("work", size, Class.CLIENT_DATA)
    a.freeze(g)
    a.write(work, 0, np.zeros(size, np.uint8))
    for c, q, q_heads, lens, s, arrays, out in keep:
        for k, v in arrays.items():
            a.write(s[k], 0, v)
        kv = Kv8(a.ptr(s["codes"]), a.ptr(s["scales"]), a.ptr(s["table"]), c.pool, c.kv_heads, *c.table.shape)
        calls.append(g.capture(lambda kv=kv, s=s, q_heads=q_heads, out=out: g.kv8_attention(
            kv, a.ptr(s["q"]), q_heads, a.ptr(s["lens"]), a.ptr(out), 0.088, a.ptr(work), size)))
    for i in (0, 1, 2, 1, 0, 2, 2, 0, 1):
        g.launch_graph(calls[i])
    g.sync()
    for c, q, q_heads, lens, s, arrays, out in keep:
        got = a.read_array(out, 0, q.size, np.uint16).reshape(q.shape)
        assert (got == kernels.kv8_attention(c, q, q_heads, lens, scale=0.088)).all()
        check_attention(c, q, q_heads, lens, got, scale=0.088)


def test_calls_without_work(kernels):
    """No rows, no sequences: nothing is launched, nothing is written."""
    rng = np.random.default_rng(20)
    c = R.fill(rng, 2, [20], 3)
    qn, kn = norm_weights(rng)
    launches = kernels.gpu.counts()["launches"]
    q, after, _ = kernels.kv8_write(c, np.zeros((0, 8 * HEAD), np.uint16), 4, qn, kn, THETA, EPS, 48, [], [])
    assert q.size == 0 and (after.codes == c.codes).all()
    none = type(c)(c.codes, c.scales, np.zeros((0, 3), np.uint32))
    assert kernels.kv8_attention(none, np.zeros((0, 4, HEAD), np.uint16), 4, []).size == 0
    assert kernels.kv8_select(none, R.all_bounds(c), np.zeros((0, 4, HEAD), np.uint16), 4, [], 3).size == 0
    k, _ = kernels.kv8_read(none, [], np.zeros((0, 3), np.uint32), 2)
    assert (k == kernels.SENTINEL).all()
    assert kernels.gpu.counts()["launches"] == launches + 1  # the rope table's


def test_calls_of_all_sizes_share_a_workspace(kernels):
    """Selection and attention of one sequence and of batches in turn over one workspace, twice: the numbers of
    sequences and heads change what lies in it, the results do not."""
    from x0ne_core import Arena, Kv8
    from x0ne_core.arena import Class
    rng = np.random.default_rng(21)
    g, a, keep, budget = kernels.gpu, Arena(), [], 4
    shapes = [(8, 16, [4000]), (8, 8, [1500] * 20 + [300]), (1, 2, [2100, 40]), (3, 3, [1300] * 50), (1, 16, [0])]
    size = 0
    for kvh, q_heads, lens in shapes:
        c = R.fill(rng, kvh, [min(n, 1300) for n in lens[:3]], 260)
        table = np.resize(c.table, (len(lens), 260))  # more sequences of the same pages
        c = type(c)(c.codes, c.scales, table)
        q = random_q(rng, len(lens), q_heads)
        lens = [min(n, 1300) for n in lens]
        size = max(size, g.kv8_work_bytes(Kv8(16, 16, 16, c.pool, kvh, *table.shape), q_heads))
        arrays = {"codes": c.codes, "scales": c.scales, "table": table, "q": q, "lens": np.array(lens, np.uint32),
                  "bounds": R.all_bounds(c)}
        outs = {"out": q.nbytes, "sparse": q.nbytes, "list": len(lens) * kvh * budget * 4}
        keep.append((c, q, q_heads, lens, arrays, {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()},
                     {k: a.alloc(k, n, Class.CLIENT_DATA) for k, n in outs.items()}))
    work = a.alloc("work", size, Class.CLIENT_DATA)
    a.freeze(g)
    a.write(work, 0, np.zeros(size, np.uint8))
    for turn in range(2):
        for c, q, q_heads, lens, arrays, s, o in keep:
            for k, v in arrays.items():
                a.write(s[k], 0, v)
            for k in ("out", "sparse"):
                a.write(o[k], 0, np.full(q.size, kernels.SENTINEL, np.uint16))
            kv = Kv8(a.ptr(s["codes"]), a.ptr(s["scales"]), a.ptr(s["table"]), c.pool, c.kv_heads, *c.table.shape)
            g.kv8_select(kv, a.ptr(s["bounds"]), a.ptr(s["q"]), q_heads, a.ptr(s["lens"]), budget, a.ptr(o["list"]), a.ptr(work), size)
            g.kv8_attention(kv, a.ptr(s["q"]), q_heads, a.ptr(s["lens"]), a.ptr(o["out"]), 0.088, a.ptr(work), size)
            g.kv8_attention(kv, a.ptr(s["q"]), q_heads, a.ptr(s["lens"]), a.ptr(o["sparse"]), 0.088, a.ptr(work), size,
                            page_list=a.ptr(o["list"]), budget=budget)
            g.sync()
            pages = a.read_array(o["list"], 0, len(lens) * c.kv_heads * budget, np.uint32).reshape(len(lens), c.kv_heads, budget)
            assert (pages == R.select(c, arrays["bounds"], vals(q), lens, budget)).all(), (turn, len(lens))
            check_attention(c, q, q_heads, lens, a.read_array(o["out"], 0, q.size, np.uint16), scale=0.088)
            check_attention(c, q, q_heads, lens, a.read_array(o["sparse"], 0, q.size, np.uint16), page_list=pages, scale=0.088)


def test_more_pairs_than_counters(kernels):
    """1024 kv heads by 130 sequences are three launches (65536 pairs each at most): every sequence's pages and output
    those of its twin, whose table, queries and length it shares, and the twins' those of the plain form."""
    rng = np.random.default_rng(22)
    kvh, seq_pages, budget, n = 1024, 68, 3, 130
    lens = [1070, 25, 0, 1088]
    c = R.empty(6, kvh, 4, 1)
    x = vals(bits(rng.standard_normal((2, 6 * PAGE, kvh, HEAD))))
    (kc, ks), (vc, vs) = R.quantise(x[0]), R.quantise(x[1])
    split = lambda b: b.reshape(6, PAGE, kvh, *b.shape[2:])
    c.codes[:, :, :2048] = split(kc).transpose(0, 2, 1, 3).reshape(6, kvh, 2048)
    c.codes[:, :, 2048:] = split(vc).transpose(0, 2, 3, 1).reshape(6, kvh, 2048)
    c.scales[:, :, :PAGE], c.scales[:, :, PAGE:] = split(ks).transpose(0, 2, 1), split(vs).transpose(0, 2, 1)
    four = rng.integers(0, 6, (4, seq_pages)).astype(np.uint32)
    q4 = random_q(rng, 4, kvh).reshape(4, kvh, HEAD)
    of = np.arange(n) % 4
    c = type(c)(c.codes, c.scales, four[of])
    launches = kernels.gpu.counts()["launches"]
    pages = kernels.kv8_select(c, R.all_bounds(c), q4[of], kvh, np.array(lens)[of], budget)
    out = kernels.kv8_attention(c, q4[of], kvh, np.array(lens)[of])
    assert kernels.gpu.counts()["launches"] == launches + 6
    assert (pages == pages[:4][of]).all() and (out == out[:4][of]).all()
    some = [0, 1, 510, 1023]
    few = type(c)(c.codes[:, some], c.scales[:, some], four)
    assert (pages[:4, some] == R.select(few, R.all_bounds(few), vals(q4[:, some]), lens, budget)).all()
    check_attention(few, q4[:, some], 4, lens, out[:4, some])


def test_two_gpus_streams_at_once(kernels):
    """Two Gpus of one device, each with its stream and workspace, their calls issued in turn without a wait between:
    each the bits it has alone."""
    from x0ne_core import Arena, Gpu, Kv8
    from x0ne_core.arena import Class
    rng = np.random.default_rng(24)
    pairs = []
    for g, (kvh, q_heads, lens) in zip((kernels.gpu, Gpu()), [(8, 32, [6000, 50, 0]), (2, 8, [3000] * 9)]):
        c = R.fill(rng, kvh, lens, 376)
        q, a, budget = random_q(rng, len(lens), q_heads), Arena(), 9
        size = g.kv8_work_bytes(Kv8(16, 16, 16, c.pool, kvh, *c.table.shape), q_heads)
        bounds = R.all_bounds(c)
        arrays = {"codes": c.codes, "scales": c.scales, "table": c.table, "q": q, "lens": np.array(lens, np.uint32),
                  "bounds": bounds, "work": np.zeros(size, np.uint8)}
        s = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()}
        s.update({k: a.alloc(k, n, Class.CLIENT_DATA) for k, n in
                  {"out": q.nbytes, "sparse": q.nbytes, "list": len(lens) * kvh * budget * 4}.items()})
        a.freeze(g)
        for k, v in arrays.items():
            a.write(s[k], 0, v)
        at = {k: a.ptr(v) for k, v in s.items()}
        pairs.append((g, c, q, q_heads, lens, bounds, budget, size, a, s, at, Kv8(at["codes"], at["scales"], at["table"], c.pool, kvh, *c.table.shape)))
    for _ in range(10):
        for g, c, q, q_heads, lens, bounds, budget, size, a, s, at, kv in pairs:
            g.kv8_select(kv, at["bounds"], at["q"], q_heads, at["lens"], budget, at["list"], at["work"], size)
            g.kv8_attention(kv, at["q"], q_heads, at["lens"], at["out"], 0.088, at["work"], size)
            g.kv8_attention(kv, at["q"], q_heads, at["lens"], at["sparse"], 0.088, at["work"], size, page_list=at["list"], budget=budget)
    for g, *_ in pairs:
        g.sync()
    for g, c, q, q_heads, lens, bounds, budget, size, a, s, at, kv in pairs:
        read = lambda k, n, t: a.read_array(s[k], 0, n, t)
        pages = read("list", len(lens) * c.kv_heads * budget, np.uint32).reshape(len(lens), c.kv_heads, budget)
        assert (pages == kernels.kv8_select(c, bounds, q, q_heads, lens, budget)).all()
        assert (read("out", q.size, np.uint16).reshape(q.shape) == kernels.kv8_attention(c, q, q_heads, lens, scale=0.088)).all()
        assert (read("sparse", q.size, np.uint16).reshape(q.shape) ==
                kernels.kv8_attention(c, q, q_heads, lens, page_list=pages, scale=0.088)).all()
