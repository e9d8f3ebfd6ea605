"""A Gpu is closed while a capture of another is open: its memory comes back, the capture stays whole, and no error is left
behind for a later launch."""
import ctypes as C
import threading

import numpy as np
import pytest

from w4_reference import bits

pytestmark = pytest.mark.gpu

ROWS, COLS, N = 512, 4096, 40  # a bf16 product in K slices, whose Gpu takes its 64 MiB workspace


def product(gpu, rng):
    """An arena with a product's operands, a call of it, and its result."""
    from x0ne_core import Arena
    from x0ne_core.arena import Class
    a = Arena()
    need = {"w": bits(rng.standard_normal((ROWS, COLS)) * 0.02), "x": bits(rng.standard_normal((N, COLS)))}
    sl = {k: a.alloc(k, v.nbytes, Class.CLIENT_DATA) for k, v in need.items()} | {"y": a.alloc("y", N * ROWS * 4, Class.CLIENT_DATA)}
    a.freeze(gpu)
    for k, v in need.items():
        a.write(sl[k], 0, v)
    at = {k: a.ptr(v) for k, v in sl.items()}

    def result(clear=False):
        gpu.sync()
        y = a.read_array(sl["y"], 0, N * ROWS, np.uint32)
        if clear:
            a.write(sl["y"], 0, np.zeros(N * ROWS, np.uint32))
        return y

    return a, lambda g: g.gemv(at["w"], ROWS, COLS, at["x"], N, at["y"], True), result


@pytest.mark.parametrize("same_thread", [False, True])
def test_a_gpu_is_closed_while_another_captures(kernels, same_thread):
    """One that has its workspace, and one that is made and closed inside the capture."""
    from x0ne_core import Gpu
    g = kernels.gpu
    a, call, result = product(g, np.random.default_rng(1))
    call(g)
    want = result(clear=True)
    other, third = Gpu(), Gpu()
    for gpu in (other, third):
        call(gpu)
        gpu.sync()
    result(clear=True)
    before = g.mem_info()[0]
    errors = []

    def closes():
        try:
            other.close()
            call(third)  # its launches look at this thread's last error
            fresh = Gpu()
            fresh.close()
            call(third)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    def captured():
        call(g)
        if same_thread:
            closes()
        else:
            t = threading.Thread(target=closes)
            t.start()
            t.join()
        call(g)

    graph = g.capture(captured)
    assert not errors, errors
    third.sync()
    # The workspace's 64 MiB come back or stay; the graph made in between took a few.
    freed = (g.mem_info()[0] - before) / (1 << 20)
    assert freed > 32, f"{freed} MiB more are free"
    for _ in range(3):
        result(clear=True)
        g.launch_graph(graph)
        assert (result() == want).all()
    graph.close()
    third.close()
    a.close()


def test_a_gpu_takes_no_device_memory_beside_its_stream(kernels):
    """64 of them against 64 streams of the runtime: less than 8 MiB apart, 128 KiB to each. The first turn of either makes what
    the runtime keeps."""
    from x0ne_core import Gpu, lib
    streams = []

    def stream():
        s = C.c_void_p()
        assert lib().hipStreamCreateWithFlags(C.byref(s), 1) == 0  # non-blocking, of the runtime that the library uses
        streams.append(s)

    def taken(make):
        before = kernels.gpu.mem_info()[0]
        made = [make() for _ in range(64)]
        took = (before - kernels.gpu.mem_info()[0]) / (1 << 20)
        for g in made:
            if g:
                g.close()
        while streams:
            assert lib().hipStreamDestroy(streams.pop()) == 0
        return took

    for _ in range(2):
        of_streams, of_gpus = taken(stream), taken(Gpu)
    print(f"MEASURE MiB taken by 64 streams {of_streams}, by 64 Gpus {of_gpus}")
    assert of_gpus - of_streams < 8
