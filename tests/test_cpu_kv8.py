"""The 8-bit paged K/V cache on the CPU: its host rules (kv8.h) over their whole range, the plain form the GPU tests
compare with, and every refusal, before any device is touched."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import kv8_reference as R
from common import ROOT, run_cpp


def test_the_host_rules(tmp_path):
    assert run_cpp(tmp_path, "kv8_model.cpp") == "ok\n"


def test_the_plain_form_rounds_to_the_nearest_code():
    """Every bf16 magnitude alone in a row: its code's value is the nearest of all e4m3 values under its scale, above
    half of the range unless the exponent is the lowest; what is not finite is NaN."""
    x = np.zeros((1 << 15, 128))
    x[:, 0] = R.vals(np.arange(1 << 15))
    with np.errstate(invalid="ignore"):
        codes, scales = R.quantise(x)
    finite = np.isfinite(x[:, 0])
    assert (codes[~finite, 0] == 0x7F).all() and (codes[:, 1:] == 0).all()
    e = scales[finite].astype(np.float64) - 127
    y, code = x[finite, 0] / 2.0 ** e, codes[finite, 0]
    assert (y <= 448).all() and ((y > 224) | (e == R.LOWEST)).all()
    assert (np.abs(R.VALUES[code] - y) <= np.abs(R.GRID[None] - y[:, None]).min(1)).all()


def call(name, **change):
    """A valid call without a device, with some arguments changed: the error that it raises."""
    from x0ne_core import _lib
    cache = dict(codes=4096, scales=4096, page_table=4096, pool=8, kv_heads=2, seqs=3, seq_pages=4)
    args = {"write": dict(qkv=256, rows=5, q_heads=8, q_norm=256, k_norm=256, eps=1e-6, rope_cs=256, positions=64, row_seq=256,
                          row_pos=256, q_out=256, bounds=0),
            "read": dict(lens=256, k=256, v=256, out_table=256, out_pool=8),
            "attention": dict(q=256, q_heads=8, lens=256, page_list=0, budget=0, out=256, scale=0.1, work=256, work_bytes=1 << 40),
            "select": dict(bounds=256, q=256, q_heads=8, lens=256, budget=4, page_list=256, work=256, work_bytes=1 << 40)}[name]
    for k, v in change.items():
        (cache if k in cache else args)[k] = v
    c = _lib.Kv8C(**cache)
    f = getattr(_lib.lib(), f"x0ne_gpu_kv8_{name}")
    status = f(None, None if change.get("cache", 1) is None else C.byref(c), *(v for k, v in args.items() if k != "cache"))
    return status, _lib.last_error()


REFUSED = {
    "": [dict(codes=0), dict(codes=4104), dict(scales=0), dict(scales=4100), dict(page_table=0), dict(page_table=4097),
         dict(pool=0), dict(kv_heads=0), dict(kv_heads=1025), dict(seqs=65536), dict(seq_pages=0), dict(seq_pages=1 << 24),
         dict(cache=None)],
    "write": [dict(qkv=0), dict(qkv=258), dict(q_norm=0), dict(q_norm=264), dict(k_norm=0), dict(k_norm=264), dict(rope_cs=0),
              dict(rope_cs=264), dict(row_seq=0), dict(row_seq=258), dict(row_pos=0), dict(row_pos=258), dict(q_out=0),
              dict(q_out=264), dict(bounds=264), dict(q_heads=0), dict(q_heads=16385), dict(rows=1 << 24), dict(rows=1 << 63)],
    "read": [dict(lens=0), dict(lens=258), dict(k=0), dict(k=264), dict(v=0), dict(v=264), dict(out_table=0),
             dict(out_table=258), dict(out_pool=0)],
    "attention": [dict(q=0), dict(q=264), dict(lens=0), dict(lens=258), dict(out=0), dict(out=264), dict(q_heads=0),
                  dict(q_heads=7), dict(q_heads=34), dict(page_list=256), dict(budget=4), dict(page_list=258, budget=4),
                  dict(page_list=256, budget=1 << 24), dict(work=0), dict(work=128), dict(work_bytes=255)],
    "select": [dict(bounds=0), dict(bounds=264), dict(q=0), dict(q=264), dict(lens=0), dict(lens=258), dict(page_list=0),
               dict(page_list=258), dict(budget=0), dict(budget=1 << 24), dict(q_heads=0), dict(q_heads=7), dict(q_heads=34),
               dict(work=0), dict(work=128), dict(work_bytes=255), dict(seq_pages=65535 * 64 + 1, work_bytes=1 << 60)],
}


@pytest.mark.parametrize("name", ["write", "read", "attention", "select"])
def test_refusals_come_before_any_device(name):
    from x0ne_core import _lib
    for change in REFUSED[""] + REFUSED[name]:
        status, message = call(name, **change)
        assert status == _lib.ERR_FORMAT and message.startswith(f"kv8 {name}: "), (change, status, message)
    assert call(name)[0] == _lib.ERR_GPU  # as asked, and no device


def test_the_workspace_size():
    from x0ne_core import _lib
    f = _lib.lib().x0ne_kv8_work_bytes
    ok = dict(codes=16, scales=16, page_table=16, pool=8, kv_heads=2, seqs=3, seq_pages=4)
    assert f(C.byref(_lib.Kv8C(**ok)), 8) >= 256
    assert f(None, 8) == 0 and f(C.byref(_lib.Kv8C(**ok)), 7) == 0 and f(C.byref(_lib.Kv8C(**{**ok, "pool": 0})), 8) == 0
    big = f(C.byref(_lib.Kv8C(**{**ok, "kv_heads": 1024, "seqs": 65535, "seq_pages": (1 << 24) - 1})), 16384)
    assert 65535 * 1024 * ((1 << 24) - 1) * 8 <= big < 1 << 63


def test_the_rust_and_python_structs_are_the_headers():
    from x0ne_core._lib import Kv8C
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "x0ne_core.h")).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\}\s*x0ne_kv8;", header).group(1)
    fields = [(name.strip(), kind) for kind, names in re.findall(r"(uint\d+_t)\s+([^;]+);", body) for name in names.split(",")]
    rust = open(os.path.join(ROOT, "x0ne-engine_amd", "rust", "x0ne-core-runtime-mi355x", "src", "sys.rs")).read()
    m = re.search(r"#\[repr\(C\)\]\s*#\[derive\([^)]*\)\]\s*pub struct x0ne_kv8 \{(.*?)\}", rust, re.S)
    assert re.findall(r"pub (\w+): (\w+)", m.group(1)) == [(n, {"uint64_t": "u64", "uint32_t": "u32"}[k]) for n, k in fields]
    assert Kv8C._fields_ == [(n, {"uint64_t": C.c_uint64, "uint32_t": C.c_uint32}[k]) for n, k in fields]
    for name in re.findall(r"\b(x0ne_\w*kv8_\w+)\s*\(", header):
        assert f"pub fn {name}(" in rust, name


def test_caches_of_all_shapes_have_their_counters_in_the_same_place():
    """What a call leaves behind its counters may not lie where a call of another cache counts: the part of the
    workspace in front of the states (of 132 floats a slice) and scores (8 bytes a page) is the same for all."""
    from x0ne_core import _lib
    f = _lib.lib().x0ne_kv8_work_bytes
    for kv_heads, seqs in [(1, 1), (8, 1), (8, 16), (8, 64), (2, 700), (1024, 64)]:
        size = [f(C.byref(_lib.Kv8C(16, 16, 16, 8, kv_heads, seqs, pages)), kv_heads) for pages in (1 << 20, 1 << 21)]
        assert size[0] - (size[1] - size[0]) == 4 * 65536, (kv_heads, seqs, size)


def test_the_workspace_is_sized_before_the_cache_has_addresses():
    from x0ne_core import _lib
    f, numbers = _lib.lib().x0ne_kv8_work_bytes, (8, 2, 3, 4)
    assert f(C.byref(_lib.Kv8C(0, 0, 0, *numbers)), 8) == f(C.byref(_lib.Kv8C(4096, 4096, 4096, *numbers)), 8) > 4 * 65536
    for refused in [(0, 2, 3, 4), (8, 0, 3, 4), (8, 1025, 3, 4), (8, 2, 65536, 4), (8, 2, 3, 0), (8, 2, 3, 1 << 24)]:
        assert f(C.byref(_lib.Kv8C(0, 0, 0, *refused)), 8) == 0, refused
