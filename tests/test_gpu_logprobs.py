"""Log probabilities of logits (x0ne_gpu_logprobs) against their plain 64-bit form (w4_reference.py): ids exactly, numbers
within a derived tolerance; the chain from a row of a 4-bit head; graphs; workspaces shared with the 8-bit cache."""
import numpy as np
import pytest

import w4_reference as R
from w4_reference import NONE, bits, vals

pytestmark = pytest.mark.gpu


def check(kernels, x, tokens=None, top=0, scale=1.0, vocab=None, calls=1):
    """x [rows][stride]: f32 logits or bf16 bits.
    With M the largest |scale l| among the logits that count (within 120 of the largest): a difference from the largest is
    3 roundings of M or its own 2 M off, an exponential 2 M + 2 more, a sum of them at most 64 roundings (16 of a lane, the
    rest in trees), the logarithm 2: 64 + 8 M units of 2^-24 on a log probability, beside its own roundings where it is far
    below. The entropy's second term is a mean of differences: each error once more times 1 + H."""
    exact = (vals(x) if x.dtype == np.uint16 else x.astype(np.float64))[:, :vocab]
    got = kernels.logprobs(x, tokens, top, True, scale, vocab, calls)
    want = R.logprobs(exact, scale, tokens, top)
    with np.errstate(invalid="ignore"):
        y = exact * scale
        near = np.where(np.isfinite(y) & (y > y.max(-1, keepdims=True) - 120.0), np.abs(y), 0.0)
    unit = ((64 + 8 * near.max(-1)) * 2.0 ** -24)
    for name, g, w in zip(("token_lp", "entropy", "top_ids", "top_lp"), got, want):
        if g is None:
            continue
        if name == "top_ids":
            assert (g == w).all(), f"{int((g != w).sum())} of the ids differ"
            continue
        tol = unit * (1 + np.abs(np.where(np.isnan(w), 0.0, w))) if name == "entropy" else \
            unit[:, None] + 2.0 ** -22 * np.abs(np.where(np.isfinite(w), w, 0.0))
        w = np.where(w <= -(2.0 ** 128), -np.inf, w)  # 3e38 below 3e38 is past f32's 2^128: -infinity is its nearest
        same = (np.isnan(g) & np.isnan(w)) | (g == w)
        with np.errstate(invalid="ignore"):
            worst = np.where(same, 0.0, np.abs(g - w) / tol)
        assert np.isfinite(worst).all() and (worst.max() if worst.size else 0.0) <= 1.0, (name, float(np.nanmax(worst)))
    return got


def logits(rng, rows, vocab, kind="f32"):
    x = rng.standard_normal((rows, vocab)) * 2.5 + 12.0 * (rng.random((rows, vocab)) < 3.0 / vocab)
    return bits(x) if kind == "bf16" else x.astype(np.float32)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 63), (2, 64), (2, 65), (4, 1000), (3, 4095), (3, 4096), (2, 4097), (2, 8193),
                                        (7, 32001), (2, 151936), (300, 777)])
def test_rows_of_all_sizes(kernels, rows, vocab, kind):
    rng = np.random.default_rng(rows + vocab)
    x = logits(rng, rows, vocab, kind)
    check(kernels, x, rng.integers(0, vocab, (rows, 3)), min(20, vocab))


@pytest.mark.parametrize("top", [0, 1, 2, 5, 20, 63, 64])
@pytest.mark.parametrize("vocab", [40, 3000, 50001])
def test_top_alternatives(kernels, top, vocab):
    """More than there are, among them; logits with many equal ones, and all equal."""
    rng = np.random.default_rng(top + vocab)
    for kind in ("f32", "bf16"):
        check(kernels, logits(rng, 3, vocab, kind), None, top)
    check(kernels, np.round(rng.standard_normal((3, vocab)) * 2).astype(np.float32), None, top)
    check(kernels, np.full((2, vocab), -3.25, np.float32), None, top)
    check(kernels, np.where(rng.random((2, vocab)) < 0.5, -0.0, 0.0).astype(np.float32), None, top)


@pytest.mark.parametrize("order", ["rising", "falling", "blocks"])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_top_alternatives_in_one_place(kernels, order, top):
    """Orders that put the largest logits into few lanes: rising and falling rows, and lanes that hold only large ones."""
    vocab = 20000
    x = np.arange(vocab, dtype=np.float32) / 1000.0
    if order == "falling":
        x = x[::-1].copy()
    if order == "blocks":
        x = np.where(np.arange(vocab) % 1024 // 4 < 100, x + 30.0, x)
        x = np.where(np.arange(vocab) % 2048 // 8 < 50, x + 1.0, x).astype(np.float32)
    check(kernels, np.stack([x, -x, x]), None, top)
    check(kernels, bits(np.stack([x, -x])), None, top)


@pytest.mark.parametrize("vocab", [300, 4096, 40000])
def test_masked_rows(kernels, vocab):
    """Masks of -infinity and of the lowest value that leave one, a few or no logits, at the ends; rows of NaN, of
    infinities, of both; an id past the vocabulary."""
    rng = np.random.default_rng(vocab)
    x = logits(rng, 14, vocab)
    low = np.finfo(np.float32).min
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2, :-1] = -np.inf
    x[3] = np.where(rng.random(vocab) < 0.99, -np.inf, x[3])
    x[4] = low
    x[5, 7:] = low
    x[6] = np.where(rng.random(vocab) < 0.9, low, x[6])
    x[7, vocab // 2] = np.nan
    x[8] = -np.inf
    x[8, vocab - 1] = np.nan
    x[9, 3] = np.inf
    x[10] = -np.inf
    x[10, 5] = np.inf
    x[11, 0], x[11, 1] = np.nan, np.inf
    x[12] = np.nan
    tokens = np.stack([np.zeros(14), np.full(14, vocab - 1), np.full(14, vocab), np.full(14, NONE), rng.integers(0, vocab, 14)], 1)
    check(kernels, x, tokens.astype(np.uint32), 10)
    check(kernels, bits(x), tokens.astype(np.uint32), 10)  # the lowest f32 rounds to -infinity


@pytest.mark.parametrize("scale", [0.25, 1.0, 1.7, 40.0])
def test_scales_and_far_logits(kernels, scale):
    rng = np.random.default_rng(3)
    x = logits(rng, 6, 9000)
    x[1] += 1000.0
    x[2] -= 1000.0
    x[3] *= 1e-3
    x[4] *= 50.0
    x[5] = 3.0e38 * np.sign(x[5])  # scale l may be past f32
    check(kernels, x, rng.integers(0, 9000, (6, 2)), 8, scale)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,stride", [(1000, 1001), (1000, 1003), (4099, 4100), (31, 64), (20001, 20480)])
def test_strides(kernels, vocab, stride, kind):
    """Padding of large values behind each row, which nothing may count."""
    rng = np.random.default_rng(stride)
    x = logits(rng, 5, stride, "f32")
    x[:, vocab:] = 1000.0
    check(kernels, bits(x) if kind == "bf16" else x, rng.integers(0, vocab, (5, 1)), 7, vocab=vocab)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 8192), (600, 8000), (300, 8192), (2, 16384), (40, 16001), (2, 16385), (256, 17000), (257, 17000), (512, 16390), (513, 16390),
                                        (1, 32768), (30, 32768), (1, 32769), (60, 50257), (62, 50001), (3, 262144), (12, 262145)])
def test_rows_cut_in_every_way(kernels, rows, vocab, kind):
    """Sizes at both sides of each rule by which rows are cut, with no, one and more alternatives; equal logits in rows that
    the floor does not part."""
    rng = np.random.default_rng(rows + vocab)
    x = logits(rng, rows, vocab, kind)
    x[0] = bits(np.full(vocab, 0.5)) if kind == "bf16" else 0.5
    x[rows // 2, :-3] = bits(np.array([-np.inf])) if kind == "bf16" else -np.inf
    tokens = rng.integers(0, vocab, (rows, 1))
    for top in (0, 1, 7):
        check(kernels, x, tokens, top)


def test_more_tokens_than_a_block_and_repeated_ones(kernels):
    rng = np.random.default_rng(8)
    tokens = rng.integers(0, 5000, (3, 1111))
    tokens[:, 5:50] = 17
    check(kernels, logits(rng, 3, 5000), tokens, 3)


def test_more_rows_than_a_launch(kernels):
    """70000 rows: two pairs of launches over one workspace, twice."""
    rng = np.random.default_rng(9)
    x = np.tile(logits(rng, 7, 4100), (10000, 1))
    got = kernels.logprobs(x, np.tile(np.arange(7)[:, None] * 500, (10000, 1)), 2, calls=2)
    want = check(kernels, x[:7], np.arange(7)[:, None] * 500, 2)
    for name, g, w in zip(("token_lp", "entropy", "top_ids", "top_lp"), got, want):
        g = g.reshape(10000, *w.shape)
        assert (g == g[:1]).all()
        # Fewer rows are cut into other slices: each within its tolerance of the exact value (M at most 30, H at most 9).
        assert (g[0] == w).all() if name == "top_ids" else (np.abs(g[0] - w) <= 2 * (64 + 8 * 30) * 10 * 2.0 ** -24).all()


def test_a_large_vocabulary(kernels):
    rng = np.random.default_rng(10)
    x = logits(rng, 2, 1 << 20)
    check(kernels, x, rng.integers(0, 1 << 20, (2, 4)), 64, calls=3)


def test_the_same_call_gives_the_same_bits(kernels):
    rng = np.random.default_rng(11)
    x, tokens = logits(rng, 9, 50000), rng.integers(0, 50000, (9, 2))
    first = check(kernels, x, tokens, 20)
    for a, b in zip(first, check(kernels, x, tokens, 20, calls=6)):
        assert (a == b).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_past_32_bits(kernels, kind):
    """Rows 2^31 and some logits apart: the last begins behind 8 or 16 GiB."""
    from x0ne_core import Arena, LogProbs
    from x0ne_core.arena import Class
    rng = np.random.default_rng(12)
    g, vocab, stride, top = kernels.gpu, 9000, (1 << 31) + 17, 4
    x = logits(rng, 3, vocab, kind)
    a, size = Arena(), g.logprobs_work_bytes(LogProbs(rows=3, vocab=vocab, top=top))
    need = {"x": (2 * stride + vocab) * x.itemsize, "work": size, "ids": 3 * top * 4, "lp": 3 * top * 4, "tokens": 12, "token_lp": 12}
    sl = {k: a.alloc(k, v, Class.CLIENT_DATA) for k, v in need.items()}
    a.freeze(g)
    at = {k: a.ptr(v) for k, v in sl.items()}
    for r in range(3):
        a.write(sl["x"], r * stride * x.itemsize, x[r])
    tokens = np.array([0, 4500, 8999], np.uint32)
    a.write(sl["tokens"], 0, tokens)
    g.logprobs(LogProbs(logits=at["x"], stride=stride, tokens=at["tokens"], token_lp=at["token_lp"], top_ids=at["ids"], top_lp=at["lp"],
                        work=at["work"], work_bytes=size, rows=3, vocab=vocab, per_row=1, top=top, bf16=int(kind == "bf16")))
    g.sync()
    same = kernels.logprobs(x, tokens[:, None], top)
    assert (a.read_array(sl["token_lp"], 0, 3, np.float32) == same[0][:, 0]).all()
    assert (a.read_array(sl["ids"], 0, 3 * top, np.uint32).reshape(3, top) == same[2]).all()
    assert (a.read_array(sl["lp"], 0, 3 * top, np.float32).reshape(3, top) == same[3]).all()


# -- as they are used together --

def head(rng, vocab, hidden, group, n):
    """A 4-bit head and rows for it: arrays of a decode step's end."""
    code, s = R.quantise(vals(bits(rng.standard_normal((vocab, hidden)) * 0.05)), group)
    codes, scales = R.lay(code, s)
    return codes, scales, R.values(code, s)[:vocab, :hidden], bits(rng.standard_normal((n, hidden)))


@pytest.mark.parametrize("n", [1, 5])
def test_a_step_from_the_head_to_its_log_probabilities_in_a_graph(kernels, n):
    """Quantise, the head's product into f32 logits, log probabilities: eagerly and as a captured graph, replayed with new
    rows between eager calls of another shape over the same workspace."""
    from x0ne_core import Arena, LogProbs, W4
    from x0ne_core.arena import Class
    rng = np.random.default_rng(n)
    vocab, hidden, top, g = 9001, 512, 6, kernels.gpu
    w = bits(rng.standard_normal((vocab, hidden)) * 0.05)
    code, s = R.quantise(vals(w), 64)
    held = R.values(code, s)[:vocab, :hidden]
    d = W4(0, 0, vocab, hidden, 64)
    other = logits(rng, 3, 20000)
    size = max(g.logprobs_work_bytes(LogProbs(rows=n, vocab=vocab, top=top)), g.logprobs_work_bytes(LogProbs(rows=3, vocab=20000, top=64)))
    a = Arena()
    need = {"w": w.nbytes, "codes": d.code_bytes(), "scales": d.scale_bytes(), "x": n * hidden * 2, "logits": n * vocab * 4,
            "tokens": n * 4, "token_lp": n * 4, "entropy": n * 4, "ids": n * top * 4, "lp": n * top * 4, "work": size,
            "other": other.nbytes, "other_ids": 3 * 64 * 4, "other_lp": 3 * 64 * 4}
    sl = {k: a.alloc(k, v, Class.CLIENT_DATA) for k, v in need.items()}
    a.freeze(g)
    at = {k: a.ptr(v) for k, v in sl.items()}
    a.write(sl["w"], 0, w)
    a.write(sl["work"], 0, np.zeros(size, np.uint8))
    a.write(sl["other"], 0, other)
    d = W4(at["codes"], at["scales"], vocab, hidden, 64)
    lp = LogProbs(logits=at["logits"], stride=vocab, tokens=at["tokens"], token_lp=at["token_lp"], entropy=at["entropy"],
                  top_ids=at["ids"], top_lp=at["lp"], work=at["work"], work_bytes=size, rows=n, vocab=vocab, per_row=1, top=top)
    more = LogProbs(logits=at["other"], stride=20000, top_ids=at["other_ids"], top_lp=at["other_lp"], work=at["work"], work_bytes=size,
                    rows=3, vocab=20000, top=64)

    def step():
        g.w4_gemv(d, at["x"], n, at["logits"], "f32")
        g.logprobs(lp)

    def outputs():
        g.sync()
        return (a.read_array(sl["logits"], 0, n * vocab, np.float32).reshape(n, vocab),
                a.read_array(sl["ids"], 0, n * top, np.uint32).reshape(n, top), a.read_array(sl["lp"], 0, n * top, np.float32),
                a.read_array(sl["token_lp"], 0, n, np.float32), a.read_array(sl["entropy"], 0, n, np.float32))

    g.w4_quantise(d, at["w"])
    want_other = R.logprobs(other.astype(np.float64), 1.0, None, 64)[2]
    graph = g.capture(step)
    assert graph.nodes() == 2
    for _ in range(4):
        x = bits(rng.standard_normal((n, hidden)) * 3)
        a.write(sl["x"], 0, x)
        a.write(sl["tokens"], 0, rng.integers(0, vocab, n).astype(np.uint32))
        step()
        eager = outputs()
        assert (np.abs(eager[0] - vals(x) @ held.T) <= 1e-5 * (np.abs(vals(x)) @ np.abs(held).T)).all()
        assert (eager[1] == R.logprobs(eager[0].astype(np.float64), 1.0, None, top)[2]).all()
        g.logprobs(more)
        assert (outputs() and (a.read_array(sl["other_ids"], 0, 192, np.uint32).reshape(3, 64) == want_other).all())
        a.write(sl["ids"], 0, np.zeros(n * top, np.uint32))
        a.write(sl["logits"], 0, np.zeros(n * vocab, np.float32))
        g.launch_graph(graph)
        for e, r in zip(eager, outputs()):
            assert (e == r).all()
    graph.close()


def test_a_prompt_takes_the_read_back_and_the_bf16_product(kernels):
    """Many rows: the read-back into x0ne_gpu_gemv against the 4-bit product of the same rows, whose weights differ by the
    one rounding to bf16 of the read-back (2^-8 of each)."""
    from x0ne_core import Arena, W4
    from x0ne_core.arena import Class
    rng = np.random.default_rng(4)
    rows, cols, n, g = 512, 1024, 130, kernels.gpu
    code, s = R.quantise(vals(bits(rng.standard_normal((rows, cols)) * 0.03)), 32)
    codes, scales = R.lay(code, s)
    x = bits(rng.standard_normal((n, cols)))
    a = Arena()
    need = {"codes": codes, "scales": scales, "x": x, "w": np.zeros((rows, cols), np.uint16), "y": np.zeros((n, rows), np.float32),
            "y4": np.zeros((n, rows), np.float32)}
    sl = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in need.items()}
    a.freeze(g)
    for k, v in need.items():
        a.write(sl[k], 0, v)
    at = {k: a.ptr(v) for k, v in sl.items()}
    d = W4(at["codes"], at["scales"], rows, cols, 32)
    g.w4_read(d, at["w"])
    g.gemv(at["w"], rows, cols, at["x"], n, at["y"], True)
    g.w4_gemv(d, at["x"], n, at["y4"], "f32")
    g.sync()
    y, y4 = (a.read_array(sl[k], 0, n * rows, np.float32).reshape(n, rows) for k in ("y", "y4"))
    size = np.abs(vals(x)) @ np.abs(R.values(code, s)).T
    assert (np.abs(y - y4) <= (2.0 ** -8 + 2e-5) * size).all()


def test_a_workspace_shared_with_the_8_bit_cache(kernels):
    """Attention over the cache and log probabilities in turn over one workspace."""
    import kv8_reference as K
    from x0ne_core import Arena, Kv8, LogProbs
    from x0ne_core.arena import Class
    rng = np.random.default_rng(6)
    g, heads, kvh, lens = kernels.gpu, 8, 2, np.array([3000, 700, 0, 16], np.uint32)
    c = K.fill(rng, kvh, lens.tolist(), 200)
    q = K.bits(rng.standard_normal((4, heads * 128)))
    want = kernels.kv8_attention(c, q, heads, lens)
    x = logits(rng, 5, 30000)
    want_ids = R.logprobs(x.astype(np.float64), 1.0, None, 9)[2]
    numbers = (c.pool, kvh, 4, 200)
    size = max(g.kv8_work_bytes(Kv8(0, 0, 0, *numbers), heads), g.logprobs_work_bytes(LogProbs(rows=5, vocab=30000, top=9)))
    arrays = {"codes": c.codes, "scales": c.scales, "table": c.table, "q": q, "lens": lens, "work": np.zeros(size, np.uint8),
              "out": np.zeros(want.size, np.uint16), "x": x, "ids": np.zeros((5, 9), np.uint32), "lp": np.zeros((5, 9), np.float32)}
    a = Arena()
    sl = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()}
    a.freeze(g)
    for k, v in arrays.items():
        a.write(sl[k], 0, np.ascontiguousarray(v))
    at = {k: a.ptr(v) for k, v in sl.items()}
    d = LogProbs(logits=at["x"], stride=30000, top_ids=at["ids"], top_lp=at["lp"], work=at["work"], work_bytes=size, rows=5, vocab=30000, top=9)
    for _ in range(3):
        g.kv8_attention(Kv8(at["codes"], at["scales"], at["table"], *numbers), at["q"], heads, at["lens"], at["out"],
                        float(np.float32(128.0 ** -0.5)), at["work"], size)
        g.logprobs(d)
        g.sync()
        assert (a.read_array(sl["out"], 0, want.size, np.uint16).reshape(want.shape) == want).all()
        assert (a.read_array(sl["ids"], 0, 45, np.uint32).reshape(5, 9) == want_ids).all()
