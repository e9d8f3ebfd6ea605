"""How rows of log probabilities are cut, replayed on the host, and that the GPU tests run every kernel that a cut names."""
from common import run_cpp

ROWS = [1, 2, 3, 12, 13, 30, 60, 61, 64, 192, 193, 256, 257, 512, 513, 600, 768, 769, 1024, 4096, 65536, 65537, 1 << 20, 1 << 24]
VOCABS = [1, 15, 16, 17, 300, 4095, 4096, 4097, 8000, 8192, 8193, 12000, 16384, 16385, 32000, 32768, 32769, 50257, 65536, 151936, 262145,
          1 << 20, (1 << 24) - 1, 1 << 24]
TOPS = [0, 1, 2, 5, 12, 13, 20, 24, 25, 64]


def cuts(tmp_path, shapes):
    """(threads, each, count, length, join, at once, alternatives by groups, slices of the workspace) of (rows, vocab, top, bf16)."""
    out = run_cpp(tmp_path, "logprobs_cut.cpp", "".join(" ".join(str(int(v)) for v in s) + "\n" for s in shapes))
    return [tuple(int(v) for v in line.split()) for line in out.splitlines()]


def grid():
    return [(r, v, t, b) for r in ROWS for v in VOCABS for t in TOPS for b in (0, 1)]


def test_a_cut_covers_its_rows(tmp_path):
    for (rows, vocab, top, bf16), (threads, each, count, length, join, at_once, _, room) in zip(grid(), cuts(tmp_path, grid())):
        at = (rows, vocab, top, bf16)
        assert length <= threads * each and count * length >= vocab and length % 16 == 0, at
        assert at_once >= 1 and at_once * count * threads < 1 << 32, at  # a launch's threads
        assert min(rows, at_once) * count <= room, at
        assert join == (16 if count * top > 1024 else 4), at


def kernels_of(tmp_path, shapes):
    """The slices' kernel, how it picks (0: nothing, 1: one, 16 and 32: by groups, 64: by wavefronts), and the join's."""
    used = set()
    for (rows, vocab, top, bf16), (threads, each, count, _, join, _, in_groups, _) in zip(shapes, cuts(tmp_path, shapes)):
        pick = top if top <= 1 else 64 if top > in_groups else 16 if top <= 12 else 32
        used.add(("slices", bf16, threads, each, pick, count > 1))
        if count > 1:
            # A join's keys are ranked as they are, or picked: in one turn or more, by its own 256 threads' floor.
            keys = count * top
            turns = 0 if keys <= 128 else 1 if keys <= 256 * join else 2
            used.add(("join", bf16, join if turns else 0, (16 if top <= 12 else 64) if turns and top > 1 else top and 1, turns))
    return used


def test_the_gpu_tests_reach_every_kernel_that_a_cut_names(tmp_path):
    from test_gpu_logprobs_edges import CASES
    used = kernels_of(tmp_path, [s for s in grid() if s[0] * s[1] <= 1 << 24])
    tested = kernels_of(tmp_path, [(rows, vocab, top, bf16) for rows, vocab, tops in CASES for top in tops for bf16 in (0, 1)])
    assert used <= tested, sorted(used - tested)
