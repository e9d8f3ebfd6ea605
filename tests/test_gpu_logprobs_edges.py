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
