"""Weights in 4 bits (x0ne_gpu_w4_*) against their plain 64-bit form (w4_reference.py): codes, scales and the read-back
bit for bit, products within a derived tolerance, and bit for bit where every sum is exact."""
import numpy as np
import pytest

import w4_reference as R
from w4_reference import bits, vals

pytestmark = pytest.mark.gpu


def trained(rng, rows, cols):
    """Weights of uneven rows and a few far values."""
    w = rng.standard_normal((rows, cols)) * 0.02 * (0.5 + rng.random((rows, 1)))
    return bits(np.where(rng.random((rows, cols)) < 0.002, 8.0 * w, w))


# -- the form --

def check_form(kernels, w, group):
    rows, cols = w.shape
    code, s = R.quantise(vals(w), group)
    want_codes, want_scales = R.lay(code, s)
    codes, scales = kernels.w4_quantise(w, group)
    bad = np.isnan(vals(want_scales))
    assert (np.isnan(vals(scales)) == bad).all() and (scales[~bad] == want_scales[~bad]).all()
    # A zero's sign is not stated.
    flat = lambda c: np.stack([np.where(h == 8, 0, h) for h in (c & 15, c >> 4)])
    assert (flat(codes) == flat(want_codes)).all(), f"{int((flat(codes) != flat(want_codes)).sum())} codes differ"
    got, want = kernels.w4_read(codes, scales, rows, cols, group), R.values(code, s)[:rows, :cols]
    nan = np.isnan(want)
    assert (np.isnan(vals(got)) == nan).all() and (vals(got)[~nan] == vals(bits(want))[~nan]).all()
    return codes, scales


@pytest.mark.parametrize("rows,cols", [(1, 8), (16, 128), (15, 120), (17, 136), (33, 1000), (1000, 1096), (70, 2056)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_matrices_of_all_sizes(kernels, rows, cols, group):
    check_form(kernels, trained(np.random.default_rng(rows + cols + group), rows, cols), group)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_of_all_sizes(kernels, group):
    """Every bf16 pattern, infinities and NaN among them, in groups of its own size and in groups of all sizes; groups of
    zeros of both signs; the smallest and the largest."""
    rng = np.random.default_rng(group)
    every = np.arange(1 << 16).astype(np.uint16).reshape(256, 256)
    check_form(kernels, every, group)
    check_form(kernels, rng.permutation(every.ravel()).reshape(256, 256), group)
    finite = every.ravel()[np.isfinite(vals(every.ravel()))]
    check_form(kernels, rng.permutation(finite)[:256 * 248].reshape(256, 248), group)
    ends = rng.choice(np.array([0, 0x8000, 1, 0x8001, 0x7F, 0x80, 0x7F7F, 0xFF7F], np.uint16), (48, 256))
    check_form(kernels, ends, group)
    check_form(kernels, np.where(rng.random((16, 256)) < 0.5, 0x8000, 0).astype(np.uint16), group)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_at_the_middles_of_codes(kernels, group):
    """Scales of 8 bits whose group's weights are middles of codes times it where those are bf16, and their neighbours."""
    rng = np.random.default_rng(group + 1)
    middles = (R.GRID[1:] + R.GRID[:-1]) / 2
    rows = []
    for s in rng.choice(np.arange(128, 256), 64, replace=False):
        row = bits(rng.choice(np.concatenate([middles, R.GRID]), 128) * s / 64).astype(np.int64) + rng.integers(-1, 2, 128)
        row = np.maximum(row, 0)
        row[::group] = bits(np.array([6.0 * s / 64]))[0]
        rows.append(row)
    w = np.array(rows).astype(np.uint16)
    check_form(kernels, np.where(rng.random(w.shape) < 0.5, w | 0x8000, w).astype(np.uint16), group)


# -- products --

def held(rng, rows, cols, group):
    """Random codes and scales of uneven size: (codes, scales as they lie, their values)."""
    code = np.zeros((-(-rows // 16) * 16, -(-cols // 128) * 128), np.int64)
    code[:rows, :cols] = rng.integers(0, 16, (rows, cols))
    s = vals(bits(np.exp(rng.standard_normal((code.shape[0], code.shape[1] // group))) * 0.01))
    return (*R.lay(code, s), R.values(code, s)[:rows, :cols])


def silu(x):
    return x / (1.0 + np.exp(-x))


def check_product(w, x, y, out, group):
    """Each f32 sum within one rounding of 2^-23 (an addition that truncates) for each addition of its longest chain: the
    32 products of an instruction and the instructions of a group, the groups of a wavefront's tiles, the wavefronts.
    Then 2^-8 for a rounding to bf16, and for SwiGLU the sums' errors through a slope of at most 1.1, and 8 roundings."""
    chain = (group + w.shape[1] // 32 + 32) * 2.0 ** -23
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    tol = chain * size
    if out == "swiglu":
        h = w.shape[0] // 2
        gate, up, dg, du = want[:, :h], want[:, h:], tol[:, :h], tol[:, h:]
        want = silu(gate) * up
        tol = 1.1 * dg * (np.abs(up) + du) + np.abs(silu(gate)) * du + 8 * 2.0 ** -24 * np.abs(want)
    if out != "f32":
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)
        y = vals(y)
    worst = (np.abs(y - want) / (tol + 1e-30)).max()
    print(f"MEASURE w4 product {w.shape} x {len(x)} {out}: worst {worst:.3f} of the tolerance")
    assert worst <= 1.0


@pytest.mark.parametrize("out", ["bf16", "f32", "swiglu"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,cols,n", [(32, 8, 1), (32, 128, 1), (96, 1000, 2), (64, 2048, 3), (160, 4104, 5), (4096, 1024, 1),
                                         (544, 640, 16), (544, 648, 17), (288, 1992, 31), (96, 1096, 33), (64, 512, 64), (96, 264, 65),
                                         (32, 136, 200)])
def test_products(kernels, rows, cols, n, group, out):
    rng = np.random.default_rng(rows + cols + n + group)
    codes, scales, w = held(rng, rows, cols, group)
    x = bits(rng.standard_normal((n, cols)) * np.where(rng.random(cols) < 0.02, 20.0, 1.0))
    check_product(w, vals(x), kernels.w4_gemv(codes, scales, rows, cols, group, x, out), out, group)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 64), (15, 4), (17, 1), (31, 16), (1000, 9), (2049, 61)])
def test_products_of_uneven_rows(kernels, rows, n, out):
    rng = np.random.default_rng(rows + n)
    codes, scales, w = held(rng, rows, 520, 64)
    x = bits(rng.standard_normal((n, 520)))
    check_product(w, vals(x), kernels.w4_gemv(codes, scales, rows, 520, 64, x, out), out, 64)


@pytest.mark.parametrize("rows,cols,n", [(5120, 25600, 16), (24576, 4096, 1), (20000, 2048, 40), (6144, 4096, 64), (1024, 16384, 7)])
def test_products_of_large_matrices(kernels, rows, cols, n):
    """A sample of the rows, and all of them against the read-back by a long f32 sum on the host."""
    rng = np.random.default_rng(rows + n)
    codes, scales, w = held(rng, rows, cols, 128)
    x = bits(rng.standard_normal((n, cols)))
    y = kernels.w4_gemv(codes, scales, rows, cols, 128, x, "f32")
    check_product(w, vals(x), y, "f32", 128)


# Rows, columns, rows of x, group: every kernel that a plan uses, at sizes of its own (test_cpu_w4.py).
EXACT = [(32, 8, 1, 32), (2080, 640, 3, 128), (16416, 136, 2, 32), (70000, 256, 3, 32),  # 4 wavefronts
         (64, 4104, 2, 64), (6176, 2056, 4, 32),  # 8
         (96, 8200, 1, 32), (1024, 8264, 3, 64), (16, 25600, 1, 128),  # 16
         (96, 1160, 5, 32), (6176, 136, 8, 64), (8224, 392, 7, 128), (64, 6152, 8, 32), (16416, 640, 6, 64), (16, 25600, 5, 32),
         (96, 648, 16, 32), (6176, 200, 12, 32), (8224, 264, 16, 64), (160, 6280, 11, 128), (16448, 1032, 9, 32),
         (544, 2000, 23, 32), (96, 264, 64, 64), (8224, 328, 20, 128), (64, 6152, 45, 32), (16416, 520, 33, 64), (128, 8200, 70, 64),
         (4128, 6152, 96, 128), (96, 136, 600, 64), (33, 6152, 130, 32),
         (33056, 264, 12, 64), (16416, 264, 20, 128), (33030, 136, 40, 32)]


@pytest.mark.parametrize("rows,cols,n,group", EXACT)
def test_products_whose_sums_are_exact(kernels, rows, cols, n, group):
    """Whole x up to 7, codes whole multiples of .5 and scales 1, 2 and 4: every sum is exact in f32 (below 2^24 halves),
    so that each weight, scale and x shows in its place. SwiGLU of them: one rounding to bf16, and 8 of f32."""
    rng = np.random.default_rng(rows + cols + n)
    code = np.zeros((-(-rows // 16) * 16, -(-cols // 128) * 128), np.int64)
    code[:rows, :cols] = rng.integers(0, 16, (rows, cols))
    s = 2.0 ** rng.integers(0, 3, (code.shape[0], code.shape[1] // group))
    x = rng.integers(-7, 8, (n, cols)).astype(np.float64)
    assert 7 * 6 * 4 * 2 * cols < 1 << 24
    codes, scales = R.lay(code, s)
    want = x @ R.values(code, s)[:rows, :cols].T
    y = kernels.w4_gemv(codes, scales, rows, cols, group, bits(x), "f32", calls=2)
    assert (y == want).all()
    assert (kernels.w4_gemv(codes, scales, rows, cols, group, bits(x), "bf16") == bits(want)).all()
    if rows % 32 == 0:
        gate, up = want[:, :rows // 2], want[:, rows // 2:]
        y = vals(kernels.w4_gemv(codes, scales, rows, cols, group, bits(x), "swiglu"))
        with np.errstate(over="ignore"):
            want = silu(gate) * up
        # An exponential below 2^-126 is off by half of f32's least step, 2^-149.
        assert (np.abs(y - want) <= (2.0 ** -8 + 8 * 2.0 ** -24) * np.abs(want) + 2.0 ** -149 * np.abs(gate * up) + 2.0 ** -134).all()


@pytest.mark.parametrize("n", [1, 6, 20, 64])
def test_infinities_and_nan_stay_in_their_rows(kernels, n):
    """A token with an infinity or NaN, a group whose scale is NaN: only their own outputs show it."""
    rng = np.random.default_rng(n)
    rows, cols = 100, 1000
    codes, scales, w = held(rng, rows, cols, 32)
    code, s = R.quantise(vals(trained(rng, rows, cols)), 32)
    s[7, 3] = np.nan
    codes, scales = R.lay(code, s)
    w = R.values(code, s)[:rows, :cols]
    x = rng.standard_normal((n, cols))
    if n > 1:
        x[n // 2, 999], x[n - 1, 0] = np.nan, np.inf
    x = vals(bits(x))
    y = kernels.w4_gemv(codes, scales, rows, cols, 32, bits(x), "f32")
    fine_rows, fine_tokens = np.arange(rows) != 7, np.isfinite(x).all(1)
    assert np.isnan(y[:, 7]).all() and np.isfinite(y[fine_tokens][:, fine_rows]).all()
    if n > 1:
        assert np.isnan(y[n // 2]).all() and not np.isfinite(y[n - 1]).any()
    check_product(w[fine_rows], x[fine_tokens], y[fine_tokens][:, fine_rows], "f32", 32)


def test_swiglu_of_far_gates(kernels):
    """Gates of -3e4 to 3e4 and -0: silu(gate) up without an infinity or NaN."""
    gates = np.array([-30000.0, -200.0, -104.0, -88.5, -50.0, -1e-3, 0.0, 1e-3, 50.0, 88.5, 200.0, 30000.0, 1.0, 2.0, 3.0, 4.0])
    code = np.zeros((32, 128), np.int64)
    code[:16, 0], code[16:, 1] = 2, 2
    codes, scales = R.lay(code, np.ones((32, 4)))
    x = np.zeros((16, 128))
    x[:, 0], x[:, 1] = gates, 1.5
    x = vals(bits(x))
    y = vals(kernels.w4_gemv(codes, scales, 32, 128, 32, bits(x), "swiglu"))
    with np.errstate(over="ignore"):
        want = silu(x[:, 0]) * 1.5
    assert (np.abs(y - want[:, None]) <= (2.0 ** -8 + 8 * 2.0 ** -24) * np.abs(want)[:, None] + 2.0 ** -149 * 1.5 * np.abs(x[:, :1]) + 2.0 ** -134).all()


@pytest.mark.parametrize("rows,cols,n,out", [(4096, 1024, 1, "bf16"), (2048, 2048, 33, "swiglu")])
def test_the_same_call_gives_the_same_bits(kernels, rows, cols, n, out):
    rng = np.random.default_rng(n)
    codes, scales, _ = held(rng, rows, cols, 64)
    x = bits(rng.standard_normal((n, cols)))
    first = kernels.w4_gemv(codes, scales, rows, cols, 64, x, out)
    assert (kernels.w4_gemv(codes, scales, rows, cols, 64, x, out, calls=5) == first).all()


def test_graphs_that_share_the_workspace_of_parts(kernels):
    """Two graphs whose products leave their sums in parts, one with a bf16 product in K slices over the same workspace,
    replayed in turn with eager calls of a third shape between."""
    from x0ne_core import Arena, W4
    from x0ne_core.arena import Class
    rng = np.random.default_rng(12)
    g, shapes = kernels.gpu, [(160, 6280, 11, "f32"), (96, 8200, 45, "swiglu"), (16416, 640, 6, "bf16")]
    arrays = {}
    for i, (rows, cols, n, out) in enumerate(shapes):
        codes, scales, _ = held(rng, rows, cols, 64)
        arrays |= {f"c{i}": codes, f"s{i}": scales, f"x{i}": bits(rng.standard_normal((n, cols))), f"y{i}": np.zeros(n * rows, np.float32)}
    arrays |= {"w": bits(rng.standard_normal((512, 4096))), "x": bits(rng.standard_normal((40, 4096))), "y": np.zeros(40 * 512, np.float32)}
    a = Arena()
    sl = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in arrays.items()}
    a.freeze(g)
    for k, v in arrays.items():
        a.write(sl[k], 0, v)
    at = {k: a.ptr(v) for k, v in sl.items()}

    def call(i):
        rows, cols, n, out = shapes[i]
        g.w4_gemv(W4(at[f"c{i}"], at[f"s{i}"], rows, cols, 64), at[f"x{i}"], n, at[f"y{i}"], out)

    def sliced():
        g.gemv(at["w"], 512, 4096, at["x"], 40, at["y"], True)

    def result(k):
        g.sync()
        got = a.read_array(sl[k], 0, arrays[k].size, np.float32).copy()
        a.write(sl[k], 0, np.zeros(arrays[k].size, np.float32))
        return got

    want = {}
    for i in range(3):
        call(i)
        want[f"y{i}"] = result(f"y{i}")
    sliced()
    want["y"] = result("y")
    one, two = g.capture(lambda: (call(0), sliced())), g.capture(lambda: (call(1), call(0)))
    for _ in range(4):
        g.launch_graph(one)
        g.launch_graph(two)
        call(2)
        g.launch_graph(one)
        for k, v in want.items():
            assert (result(k).view(np.uint32) == v.view(np.uint32)).all(), k
    one.close()
    two.close()


def test_matrices_in_one_buffer_keep_to_their_own(kernels):
    """Two matrices whose codes and scales lie one behind the other, quantised and multiplied: nothing of the one shows in the
    other, and what lies behind the last stays."""
    from x0ne_core import Arena, W4
    from x0ne_core.arena import Class
    rng = np.random.default_rng(13)
    g, shapes, group = kernels.gpu, [(33, 200), (17, 136)], 32
    ws = [trained(rng, *s) for s in shapes]
    x = bits(rng.standard_normal((3, 200)))
    ds = [W4(0, 0, *s, group) for s in shapes]
    code_at, scale_at = np.cumsum([0] + [d.code_bytes() for d in ds]), np.cumsum([0] + [d.scale_bytes() for d in ds])
    a = Arena()
    need = {"codes": int(code_at[-1]) + 1024, "scales": int(scale_at[-1]) + 256, "w0": ws[0].nbytes, "w1": ws[1].nbytes, "x": x.nbytes, "y0": 3 * 33 * 4,
            "y1": 3 * 17 * 4}
    sl = {k: a.alloc(k, v, Class.CLIENT_DATA) for k, v in need.items()}
    a.freeze(g)
    at = {k: a.ptr(v) for k, v in sl.items()}
    for k in ("codes", "scales"):
        a.write(sl[k], 0, np.full(need[k], 0xA5, np.uint8))
    for i, w in enumerate(ws):
        a.write(sl[f"w{i}"], 0, w)
    a.write(sl["x"], 0, x)
    for i, s in enumerate(shapes):
        ds[i] = W4(at["codes"] + int(code_at[i]), at["scales"] + int(scale_at[i]), *s, group)
        g.w4_quantise(ds[i], at[f"w{i}"])
    g.w4_gemv(ds[0], at["x"], 3, at["y0"], "f32")
    g.w4_gemv(ds[1], at["x"], 3, at["y1"], "f32")  # its rows of x are 136 long: x as [3][136]
    g.sync()
    for i, (rows, cols) in enumerate(shapes):
        code, s = R.quantise(vals(ws[i]), group)
        xs = vals(x).ravel()[:3 * cols].reshape(3, cols)
        check_product(R.values(code, s)[:rows, :cols], xs, a.read_array(sl[f"y{i}"], 0, 3 * rows, np.float32).reshape(3, rows), "f32", group)
    for k, end in (("codes", code_at[-1]), ("scales", scale_at[-1])):
        assert (a.read_array(sl[k], 0, need[k], np.uint8)[int(end):] == 0xA5).all()


def test_two_gpus_at_once_and_one_made_in_the_others_capture(kernels):
    """Products in parts on two streams that overlap, each Gpu's counters and parts its own; the second Gpu is made while the
    first has a capture open."""
    from x0ne_core import Arena, Gpu, W4
    from x0ne_core.arena import Class
    rng = np.random.default_rng(14)
    rows, cols, n = 16416, 640, 33
    codes, scales, w = held(rng, rows, cols, 64)
    xs = [bits(rng.standard_normal((n, cols))) for _ in range(2)]
    g, made = kernels.gpu, []
    a = Arena()
    need = {"codes": codes.nbytes, "scales": scales.nbytes, "x0": xs[0].nbytes, "x1": xs[1].nbytes, "y0": n * rows * 4, "y1": n * rows * 4}
    sl = {k: a.alloc(k, v, Class.CLIENT_DATA) for k, v in need.items()}
    a.freeze(g)
    for k, v in (("codes", codes), ("scales", scales), ("x0", xs[0]), ("x1", xs[1])):
        a.write(sl[k], 0, v)
    at = {k: a.ptr(v) for k, v in sl.items()}
    d = W4(at["codes"], at["scales"], rows, cols, 64)

    def launches():
        g.w4_gemv(d, at["x0"], n, at["y0"], "f32")
        made.append(Gpu())
        g.w4_gemv(d, at["x0"], n, at["y0"], "f32")

    graph, other = g.capture(launches), made[0]
    assert graph.nodes() == 2
    for _ in range(20):
        g.launch_graph(graph)
        for _ in range(3):
            other.w4_gemv(d, at["x1"], n, at["y1"], "f32")
        g.w4_gemv(d, at["x0"], n, at["y0"], "f32")
    g.sync()
    other.sync()
    for i in range(2):
        check_product(w, vals(xs[i]), a.read_array(sl[f"y{i}"], 0, n * rows, np.float32).reshape(n, rows), "f32", 64)
    graph.close()
    other.close()


def whole(rng, rows, cols):
    """Weights that 4 bits hold as they are: codes of scale 1, a 6 in each group of 32 or more."""
    w = R.VALUES[rng.integers(0, 16, (rows, cols))]
    w[:, ::32] = 6.0
    return w


def test_a_matrix_past_32_bits(kernels):
    """Codes of more than 4 GiB and a bf16 matrix of 18: quantised, read back and multiplied, its first and last rows exactly."""
    from x0ne_core import Arena, W4
    from x0ne_core.arena import Class
    rng = np.random.default_rng(15)
    g, rows, cols, group, some = kernels.gpu, 140009, 65536, 32, 25
    d = W4(0, 0, rows, cols, group)
    assert d.code_bytes() > 1 << 32
    ends = [whole(rng, some, cols) for _ in range(2)]
    need = {"w": rows * cols * 2, "codes": d.code_bytes(), "scales": d.scale_bytes(), "x": 20 * cols * 2, "y": 20 * rows * 4}
    a = Arena()
    sl = {k: a.alloc(k, v, Class.CLIENT_DATA) for k, v in need.items()}
    a.freeze(g)
    at = {k: a.ptr(v) for k, v in sl.items()}
    d = W4(at["codes"], at["scales"], rows, cols, group)
    places = [0, (rows - some) * cols * 2]
    for w, place in zip(ends, places):
        a.write(sl["w"], place, bits(w))
    g.w4_quantise(d, at["w"])
    g.sync()
    for place in places:
        a.write(sl["w"], place, np.zeros((some, cols), np.uint16))
    g.w4_read(d, at["w"])
    g.sync()
    for w, place in zip(ends, places):
        assert (vals(a.read_array(sl["w"], place, some * cols, np.uint16).reshape(some, cols)) == w).all()
    for n in (1, 5, 20):
        x = rng.integers(-7, 8, (n, cols)).astype(np.float64)
        a.write(sl["x"], 0, bits(x))
        g.w4_gemv(d, at["x"], n, at["y"], "f32")
        g.sync()
        y = a.read_array(sl["y"], 0, n * rows, np.float32).reshape(n, rows)
        assert (y[:, :some] == x @ ends[0].T).all() and (y[:, -some:] == x @ ends[1].T).all(), n


def test_more_panels_than_a_grid(kernels):
    """65538 panels: quantised and read back in two launches, multiplied in one; every row exactly."""
    rng = np.random.default_rng(16)
    rows, cols = 65535 * 16 + 41, 8
    w = whole(rng, rows, cols)
    codes, scales = kernels.w4_quantise(bits(w), 64)
    assert (vals(kernels.w4_read(codes, scales, rows, cols, 64)) == w).all()
    for n in (1, 6, 20):
        x = rng.integers(-7, 8, (n, cols)).astype(np.float64)
        assert (kernels.w4_gemv(codes, scales, rows, cols, 64, bits(x), "f32") == x @ w.T).all(), n
