"""The shapes of tests/test_gpu_kv8_slices.py on the CPU: that the cut of decode attention (csrc/kv8.h) has their blocks
count and join slices while they hold further ones, and that their tolerances tell a missing page or key."""
import numpy as np
import pytest

import test_gpu_kv8_slices as T
from common import run_cpp
from kv8_reference import HEAD, PAGE, vals


def cuts(tmp_path, shapes):
    """Of each (kv_heads, seq_pages, budget, lengths): waves, stream, blocks, slices, counts, joins, rounds."""
    lines = [f"{kvh} {pages} {budget} {len(lens)} {' '.join(map(str, lens))}\n" for kvh, pages, budget, lens in shapes]
    return [tuple(int(x) for x in line.split()) for line in run_cpp(tmp_path, "kv8_cut.cpp", "".join(lines)).splitlines()]


def test_the_walked_shapes_join_inside_the_loop(tmp_path):
    """Every shape has more slices than blocks, counts inside the loop, and sequences that only such counts complete;
    together they are both numbers of wavefronts, the streaming loads, and every number of parts of a join."""
    got = cuts(tmp_path, [(kvh, pages, budget, [kinds[i % 4] for i in range(seqs)]) for _, kvh, kinds, seqs, pages, budget in T.WALKS])
    seen = set()
    for shape, (waves, stream, blocks, slices, counts, joins, _) in zip(T.WALKS, got):
        assert slices > blocks and counts > 0 and joins > 0, (shape, slices, blocks, counts, joins)
        quads, threads = shape[0] * HEAD // 4, 64 * waves
        seen.add((waves, stream, 4 if quads <= threads // 4 else 2 if quads <= threads // 2 else 1))
        if quads > threads:
            seen.add((waves, "twice"))
    assert seen >= {(4, 0, p) for p in (1, 2, 4)} | {(8, 1, p) for p in (1, 2, 4)} | {(8, 0, 4), (4, "twice")}, seen


def test_the_counted_shapes_are_cut_in_every_way(tmp_path):
    got = cuts(tmp_path, [(kvh, pages, 0, lens) for _, kvh, lens, pages in T.COUNTED])
    assert {w for w, *_ in got} == {4, 8} and any(s for _, s, *_ in got)
    assert any(joins for *_, joins, _ in got) and any(slices > len(lens) and not counts for (_, _, lens, _), (_, _, _, slices, counts, _, _) in zip(T.COUNTED, got))


@pytest.mark.parametrize("group,kv_heads,lens,seq_pages", T.COUNTED)
def test_a_count_tells_any_page_and_any_last_key(group, kv_heads, lens, seq_pages):
    """In each kv head: the outputs without one page, with one twice, without the last key or with one more are off by
    more than the tolerance on both sides, and with a page in another's place. (A sequence of one page has one value, which
    its mean is however often it counts.)"""
    rng = np.random.default_rng(len(lens) * 100 + kv_heads)
    c, dims = T.counting(rng, kv_heads, lens, seq_pages)
    for s, n in enumerate(lens):
        count, keys = T.counts(c, dims, s, n)
        assert count.sum() == n * kv_heads and keys.sum() == n
        for h in range(kv_heads):
            def told(change, total):
                a, b = count[h] / n, (count[h] + change) / max(total, 1)
                return (np.abs(a - b) > T.COUNT_OFF * (a + b)).any()
            unit = np.eye(HEAD)
            for p, k in enumerate(keys):
                d = dims[h, c.table[s, p]]
                assert told(-k * unit[d], n - k) and (n <= PAGE or told(k * unit[d], n + k)), (s, n, h, p)
            assert told(-unit[127], n - 1) and (n <= PAGE or n % PAGE == 0 or told(unit[127], n + 1)), (s, n, h)
            for d in range(0, 127, 9):  # one page of dim d for one of dim d + 1
                if n > 2 * PAGE and count[h][d] >= PAGE:
                    assert told(PAGE * (unit[d + 1] - unit[d]), n), (s, n, h, d)


@pytest.mark.parametrize("group,kv_heads,lens,seq_pages,rounds", T.FLAT)
def test_flat_scores_tell_any_page(tmp_path, group, kv_heads, lens, seq_pages, rounds):
    """The output of a kv head without any one page lies further from the whole one than the tolerance twice."""
    from x0ne_core.ops import attn_scale
    assert cuts(tmp_path, [(kv_heads, seq_pages, 0, lens)])[0][6] == rounds
    c, q, n = T.flat_case(group, kv_heads, lens, seq_pages)
    scale, qv = attn_scale(HEAD), vals(q).reshape(n, kv_heads, group, HEAD)
    for s in range(n):
        for h in range(kv_heads):
            k, v, w = T.flat_weights(c, qv[s, h], s, h, lens[s], scale)
            tol = T.flat_tolerance(v, w, qv[s, h], k, scale, rounds)
            whole, total = w @ v, w.sum(-1, keepdims=True)
            for p in range(-(-lens[s] // PAGE)):
                cut = slice(p * PAGE, min((p + 1) * PAGE, lens[s]))
                if cut.stop - cut.start < PAGE:  # of the last page the count tells
                    continue
                less = (whole - w[:, cut] @ v[cut]) / (total - w[:, cut].sum(-1, keepdims=True))
                assert (np.abs(less - whole / total) > 2 * tol).any(), (s, h, p)
