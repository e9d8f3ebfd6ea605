"""The shapes of tests/test_gpu_kv8_slices.py on the CPU: that the cut of decode attention (csrc/kv8.h) has their blocks
count and join slices while they hold further ones."""
import test_gpu_kv8_slices as T
from common import run_cpp
from kv8_reference import HEAD


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
