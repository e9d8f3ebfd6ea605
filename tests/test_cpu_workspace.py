"""What calls of different kinds that share a workspace agree on, without a device."""
import pytest


@pytest.mark.parametrize("kv_heads", [1, 8, 64])
def test_the_8_bit_cache_and_log_probabilities_leave_the_same_front_to_counters(kv_heads):
    """A call of no sequences, and one of no rows, needs the counters' part alone."""
    from x0ne_core import Kv8, LogProbs, _lib
    front = _lib.lib().x0ne_kv8_work_bytes(Kv8(0, 0, 0, 16, kv_heads, 0, 16), kv_heads)
    assert front >= 4 * 1024 and front % 256 == 0
    for numbers in (dict(vocab=1), dict(vocab=151936, top=64), dict(vocab=1 << 24, bf16=1)):
        assert _lib.lib().x0ne_logprobs_work_bytes(LogProbs(rows=0, **numbers)) == front, numbers
