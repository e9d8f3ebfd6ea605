"""Log probabilities at the ends of what the call takes, and through every kernel that its cut uses."""
import numpy as np
import pytest

import w4_reference as R
from test_gpu_logprobs import check, logits
from w4_reference import bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("place", [0, (1 << 24) - 1])
def test_the_largest_row_at_the_smallest_scale(kernels, place, kind):
    """2^24 logits of which one is far above: a difference times the others' sum is past f32, its share of the entropy is not."""
    x = np.full((1, 1 << 24), -80.0 * 2.0 ** 100, np.float32)
    x[0, place] = 0.0
    tokens = np.array([[place, 5]], np.uint32)
    check(kernels, bits(x) if kind == "bf16" else x, tokens, 1, 2.0 ** -100)
    x[0, :1 << 12] = 2.0 ** 98
    check(kernels, bits(x) if kind == "bf16" else x, tokens, 1, 2.0 ** -100)


# Rows, logits, alternatives: every kernel of a cut, and each way that it and the join pick (test_cpu_logprobs.py).
CASES = [(6, 4000, (0, 1, 5, 20, 64)), (6, 8000, (0, 1, 5, 20, 25, 64)), (600, 8000, (0, 1, 5, 20, 64)), (6, 12000, (0, 1, 5, 20, 25, 64)),
         (6, 30000, (0, 1, 5, 20, 25, 64)), (6, 50257, (0, 1, 5, 12, 13, 20, 64)), (66, 50257, (0, 1, 5, 12, 20, 64)),
         (6, 151936, (5, 20, 64)), (30, 151936, (0, 1, 12, 20, 64)), (6, (1 << 20) + 5, (1, 5, 12, 64)), (2, 1 << 20, (1, 5, 20, 64)),
         (1, (1 << 23) + 5000, (1, 5))]


def rows_of_all_kinds(rng, rows, vocab):
    """Row r of kind r % 6: as a head gives them, all equal, masked but for a few in one place, in quarters (many equal),
    rising, falling with a masked half."""
    x = logits(rng, rows, vocab)
    x[1::6] = -2.5
    for r in range(2, rows, 6):
        at = rng.integers(0, vocab)
        x[r, :at], x[r, at + 1 + rng.integers(0, 90):] = -np.inf, -np.inf
    x[3::6] = np.round(x[3::6] * 4) / 4
    ramp = np.arange(vocab, dtype=np.float32) / vocab * 20.0
    x[4::6] = ramp
    x[5::6] = np.where(np.arange(vocab) % 512 < 256, ramp[::-1], -np.inf)
    return x


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,tops", CASES)
def test_every_kernel_on_rows_of_all_kinds(kernels, rows, vocab, tops, kind):
    rng = np.random.default_rng(rows + vocab)
    x = rows_of_all_kinds(rng, rows, vocab)
    tokens = rng.integers(0, vocab, (rows, 1))
    for top in tops:
        check(kernels, bits(x) if kind == "bf16" else x, tokens, top)
