"""Weights in 4 bits and log probabilities on the CPU: the plain forms that the GPU tests compare with, sizes, and every
refusal, before any device is touched."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import w4_reference as R
from common import ROOT, run_cpp


# -- the plain forms --

@pytest.mark.parametrize("group", [32, 64, 128])
def test_the_plain_form_rounds_to_the_nearest_code(group):
    """Every bf16 magnitude beside every first of a group: the nearest of all values under the scale, which is within half
    a step of bf16 of the sixth of the largest."""
    rng = np.random.default_rng(group)
    x = R.vals(rng.integers(0, 0x7F80, (64, 256)).astype(np.uint16)) * rng.choice([-1.0, 1.0], (64, 256))
    x[:, ::3] = R.vals(R.bits(rng.standard_normal(x[:, ::3].shape)))
    code, s = R.quantise(x, group)
    each = np.repeat(s, group, 1)
    held = R.values(code, s)
    assert (np.abs(held - x) <= np.abs(R.VALUES[:, None, None] * each[None] - x[None]).min(0)).all()
    top = np.abs(x).reshape(64, -1, group).max(-1)
    assert (np.abs(s - top / 6) <= np.maximum(top / 6 * 2.0 ** -8, R.LEAST)).all()
    codes, scales = R.lay(code, s)
    assert codes.size == x.size // 2 and scales.size == x.size // group


def quotient_by_reciprocal(w, s):
    """The kernel's route to a code in f32: a reciprocal off by up to 2^-23 either way, a product, 15 bits of it."""
    out = []
    for off in (-1.0, 0.0, 1.0):
        inv = ((1.0 / s.astype(np.float64)) * (1.0 + off * 2.0 ** -23)).astype(np.float32)
        q = (w * inv).astype(np.float32).view(np.uint32)
        out.append(((q + np.uint32(0x80)) & np.uint32(0xFFFFFF00)).view(np.float32).astype(np.float64))
    return out


def test_a_reciprocal_gives_the_codes_of_the_quotient():
    """All 8-bit weights against all 8-bit scales over the range of binary places in which codes differ: the quotient by a
    reciprocal, rounded to 15 bits, lies on the side of every middle that the quotient does, and on it where that does."""
    middles = (R.GRID[1:] + R.GRID[:-1]) / 2
    s = np.arange(128, 256, dtype=np.float32)[None]
    for place in range(-4, 5):
        w = (np.arange(128, 256, dtype=np.float32) * np.float32(2.0 ** place))[:, None]
        exact = w.astype(np.float64) / s
        for got in quotient_by_reciprocal(w, s):
            for m in middles:
                assert (np.sign(got - m) == np.sign(w.astype(np.float64) - m * s)).all(), (place, m)


def test_the_log_probabilities_of_a_row_by_hand():
    x = np.array([[0.0, np.log(2.0), -np.inf, np.log(2.0)], [np.nan, 0, 0, 0], [-np.inf] * 4, [np.inf, 0, 0, 0]])
    lp, h, ids, best = R.logprobs(x, 1.0, np.array([[1, 4]] * 4), 4)
    assert np.allclose(lp[0, 0], np.log(0.4)) and np.isnan(lp[0, 1]) and np.allclose(h[0], -0.8 * np.log(0.4) - 0.2 * np.log(0.2))
    assert ids[0].tolist() == [1, 3, 0, R.NONE] and best[0, 3] == -np.inf
    assert np.isnan(lp[1:]).all() and np.isnan(h[1:]).all() and np.isnan(best[1:]).all() and (ids[1:] == R.NONE).all()


# -- sizes and refusals --

def w4(**change):
    from x0ne_core import _lib
    return _lib.W4C(**{**dict(codes=4096, scales=4096, rows=48, cols=256, group=32), **change})


BAD_SHAPES = [dict(rows=0), dict(rows=(1 << 24) + 1), dict(cols=0), dict(cols=12), dict(cols=(1 << 24) + 8), dict(group=0),
              dict(group=16), dict(group=48), dict(group=256), dict(rows=1 << 24, cols=(1 << 16) + 8)]
BAD_MATRICES = BAD_SHAPES + [dict(codes=0), dict(codes=4104), dict(scales=0), dict(scales=4104)]


@pytest.mark.parametrize("rows,cols,group", [(1, 8, 128), (16, 128, 64), (17, 136, 32), (151936, 4096, 128), (1 << 24, 1 << 16, 32), (1 << 16, 1 << 24, 64)])
def test_the_sizes_of_a_matrix(rows, cols, group):
    from x0ne_core import W4
    w = W4(0, 0, rows, cols, group)
    weights = -(-rows // 16) * 16 * (-(-cols // 128) * 128)
    assert w.code_bytes() == weights // 2 and w.scale_bytes() == weights // group * 2
    for change in BAD_SHAPES:
        d = W4(0, 0, **{**dict(rows=rows, cols=cols, group=group), **change})
        assert d.code_bytes() == d.scale_bytes() == 0, change


def test_w4_refusals_come_before_any_device():
    from x0ne_core import _lib
    L = _lib.lib()
    calls = {"quantise": lambda w, x=256, **k: L.x0ne_gpu_w4_quantise(None, w, x),
             "read": lambda w, x=256, **k: L.x0ne_gpu_w4_read(None, w, x),
             "gemv": lambda w, x=256, n=3, y=256, out=0: L.x0ne_gpu_w4_gemv(None, w, x, n, y, out)}
    more = {"quantise": [dict(x=0), dict(x=264)], "read": [dict(x=0), dict(x=264)],
            "gemv": [dict(x=0), dict(x=264), dict(y=0), dict(y=258), dict(out=3), dict(n=(1 << 24) + 1), dict(n=1 << 63),
                     dict(rows=16, out=2), dict(rows=40, out=2)]}
    for name, call in calls.items():
        for change in BAD_MATRICES + more[name]:
            of_call = {k: v for k, v in change.items() if k in ("x", "n", "y", "out")}
            status = call(C.byref(w4(**{k: v for k, v in change.items() if k not in of_call})), **of_call)
            assert status == _lib.ERR_FORMAT and _lib.last_error().startswith(f"w4 {name}: "), (name, change, status)
        assert call(None) == _lib.ERR_FORMAT
        assert call(C.byref(w4())) == _lib.ERR_GPU  # as asked, and no device


def asked(**change):
    from x0ne_core import _lib
    return _lib.LogProbsC(**{**dict(logits=4096, stride=1000, tokens=256, token_lp=256, entropy=256, top_ids=256, top_lp=256,
                                    work=4096, work_bytes=1 << 40, rows=3, vocab=1000, per_row=2, top=5, bf16=0, scale=1.0), **change})


BAD_NUMBERS = [dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(rows=(1 << 24) + 1), dict(top=65), dict(per_row=(1 << 24) + 1), dict(bf16=2)]


def test_logprobs_refusals_come_before_any_device():
    from x0ne_core import _lib
    f = _lib.lib().x0ne_gpu_logprobs
    for change in BAD_NUMBERS + [
            dict(logits=0), dict(logits=4098), dict(logits=4097, bf16=1), dict(stride=999), dict(stride=1 << 32), dict(scale=0.0),
            dict(scale=-1.0), dict(scale=2.0 ** -101), dict(scale=2.0 ** 101), dict(scale=float("inf")), dict(scale=float("nan")), dict(tokens=0), dict(tokens=258),
            dict(token_lp=0), dict(token_lp=258), dict(entropy=257), dict(top_ids=0), dict(top_ids=258), dict(top_lp=0),
            dict(top_lp=258), dict(work=0), dict(work=4224), dict(work_bytes=4 * 65536 - 1)]:
        status = f(None, C.byref(asked(**change)))
        assert status == _lib.ERR_FORMAT and _lib.last_error().startswith("logprobs: "), (change, status)
    assert f(None, None) == _lib.ERR_FORMAT
    for fine in [{}, dict(per_row=0, tokens=0, token_lp=0), dict(top=0, top_ids=0, top_lp=0), dict(entropy=0), dict(rows=0)]:
        assert f(None, C.byref(asked(**fine))) == _lib.ERR_GPU, fine  # as asked, and no device


def test_the_workspace_of_logprobs():
    """Room in front that is left to the counters of the 8-bit cache, as long as theirs; and enough behind it."""
    from x0ne_core import LogProbs, _lib
    size = lambda **k: _lib.lib().x0ne_logprobs_work_bytes(LogProbs(**k))
    for change in BAD_NUMBERS:
        assert size(**{**dict(rows=3, vocab=1000), **change}) == 0, change
    assert size(rows=1, vocab=1) >= 4 * 65536 and size(rows=0, vocab=5) >= 4 * 65536
    assert size(rows=512, vocab=151936, top=20) - size(rows=512, vocab=151936, top=0) >= 512 * 20 * 8
    assert size(rows=1 << 24, vocab=1 << 24, top=64) < 1 << 36


def test_a_workspace_of_logprobs_is_enough_for_less():
    """Fewer rows, logits or alternatives, of either type, need no more, whichever way their rows are cut."""
    from x0ne_core import LogProbs, _lib
    size = lambda *n: _lib.lib().x0ne_logprobs_work_bytes(LogProbs(rows=n[0], vocab=n[1], top=n[2], bf16=n[3]))
    rows = [*range(1, 130), *range(190, 300, 5), 512, 513, 768, 769, 1000, 4096, 65535, 65536, 65537, 1 << 20, 1 << 24]
    vocabs = [1, 4096, 4097, 8192, 8193, 16384, 16385, 32000, 32768, 32769, 50257, 65536, 151936, 1 << 20, (1 << 24) - 4096, 1 << 24]
    tops = [0, 1, 2, 20, 64]
    for bf16 in (0, 1):
        s = np.array([[[size(r, v, t, bf16) for t in tops] for v in vocabs] for r in rows], np.int64)
        assert all((np.diff(s, axis=k) >= 0).all() for k in range(3))
        if bf16:
            assert (s == other).all()
        other = s


def test_the_python_out_names():
    from x0ne_core import FormatError, Gpu, W4
    with pytest.raises(FormatError):
        Gpu.w4_gemv(object(), W4(), 0, 0, 0, "f64")


@pytest.mark.parametrize("name", ["x0ne_w4", "x0ne_logprobs"])
def test_the_rust_and_python_structs_are_the_headers(name):
    from x0ne_core import _lib
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "x0ne_core.h")).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\}\s*%s;" % name, header).group(1)
    fields = [(n.strip(), kind) for kind, names in re.findall(r"(uint\d+_t|float)\s+([^;]+);", body) for n in names.split(",")]
    rust = open(os.path.join(ROOT, "x0ne-engine_amd", "rust", "x0ne-core-runtime-mi355x", "src", "sys.rs")).read()
    m = re.search(r"#\[repr\(C\)\]\s*#\[derive\([^)]*\)\]\s*pub struct %s \{(.*?)\}" % name, rust, re.S)
    assert re.findall(r"pub (\w+): (\w+)", m.group(1)) == [(n, {"uint64_t": "u64", "uint32_t": "u32", "float": "f32"}[k]) for n, k in fields]
    mirror = {"x0ne_w4": _lib.W4C, "x0ne_logprobs": _lib.LogProbsC}[name]
    assert mirror._fields_ == [(n, {"uint64_t": C.c_uint64, "uint32_t": C.c_uint32, "float": C.c_float}[k]) for n, k in fields]
    for call in re.findall(r"\b(x0ne_\w*(?:w4|logprobs)\w*)\s*\(", header):
        assert f"pub fn {call}(" in rust, call


# -- how a launch is cut --

def plans(tmp_path, shapes):
    """(xl, panels, waves, even, units, rounds, groups, run, blocks, rows at once) of (rows, cols, n, swiglu, parts)."""
    out = run_cpp(tmp_path, "w4_plan.cpp", "".join(" ".join(str(int(v)) for v in s) + "\n" for s in shapes))
    return [tuple(int(v) for v in line.split()) for line in out.splitlines()]


def test_a_plan_covers_its_matrix(tmp_path):
    """Over sizes to the largest: every panel, tile and row of X is some block's, the blocks' runs are all the rounds, a unit
    a block unless they are even, and grids, counters and parts are within what there is."""
    sizes = [1, 15, 16, 17, 100, 1000, 4096, 4104, 6144, 12288, 24576, 51200, 151936, 1 << 20, 1 << 24]
    shapes = [(r, max(8, c // 8 * 8), n, s, p) for r in sizes for c in sizes for n in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 96, 200, 512)
              for s in (0, 1) for p in (0, 1) if r * c <= 1 << 40 and not (s and r % 32)]
    for (rows, cols, n, swiglu, parts), (xl, panels, waves, even, units, rounds, groups, run, blocks, most) in zip(shapes, plans(tmp_path, shapes)):
        at = (rows, cols, n, swiglu, parts)
        assert 1 <= most <= 512 and most * cols * 2 < 1 << 32 and (most == 512 or most % 32 == 0), at
        if n > most:
            continue
        tiles = -(-cols // 128)
        assert units * panels >= -(-rows // 16) > (units - 1) * panels and rounds * waves >= tiles > (rounds - 1) * waves, at
        assert groups * 4 * xl >= n > (groups - 1) * 4 * xl and not (swiglu and panels % 2), at
        assert blocks * run >= units * rounds > (blocks - 1) * run and units * rounds < 1 << 32, at
        assert -(-blocks // 8) * 8 * groups * 64 * waves < 1 << 32, at
        if even:
            tokens = -(-xl // 4)
            assert parts and units * groups <= 65536 and blocks * groups * 2 * panels * tokens * 1024 <= 64 << 20, at
            assert blocks * groups <= 256 or blocks == 1, at
        else:
            assert run == rounds and blocks == units, at


def kernels_of(tmp_path, shapes):
    return {(bool(s[3]),) + p[:4] for s, p in zip(shapes, plans(tmp_path, shapes))}


def test_the_gpu_tests_reach_every_kernel_that_a_plan_uses(tmp_path):
    """Those of the projections of the Qwen3 shapes and of a grid of others, for one row to 128, are among those of the exact
    sums' test, for which there is a kernel each."""
    from bench import QWEN3_0_6B, QWEN3_8B, QWEN3_32B
    from test_gpu_w4 import EXACT
    sizes = [16, 64, 256, 1000, 2048, 4096, 8192, 16384, 32768, 65536]
    shapes = [(r, c, n) for r in sizes for c in sizes for n in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128)]
    for m in (QWEN3_0_6B, QWEN3_8B, QWEN3_32B):
        h, i, d = m["hidden_size"], m["intermediate_size"], m["head_dim"]
        q, kv = m["num_attention_heads"] * d, m["num_key_value_heads"] * d
        shapes += [(r, c, n) for r, c in ((q + 2 * kv, h), (h, q), (2 * i, h), (h, i), (m["vocab_size"], h)) for n in range(1, 129)]
    used = kernels_of(tmp_path, [(*s, swiglu, 1) for s in shapes for swiglu in (0, 1) if not (swiglu and s[0] % 32)])
    tested = kernels_of(tmp_path, [(rows, cols, n, swiglu, 1) for rows, cols, n, _ in EXACT for swiglu in (0, 1) if not (swiglu and rows % 32)])
    assert used <= tested, used - tested
