"""What b2_lm_sync tells whom, and tile kernels whose waits run out."""
import ctypes as C
import os
import subprocess
import time

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_stream_is_told_once(native):
    """The kernels' count only grows; a stream that asks is told of whatever it has not been told, whoever asked before."""
    host = C.CDLL(native.HOST_LIB)
    asks = [(0, 1, 0, 0), (0, 2, 0, 0), (0, 1, 3, 1), (0, 2, 3, 1), (0, 1, 3, 0), (0, 2, 3, 0),  # one's question does not take the other's answer
            (0, 9, 3, 1), (1, 1, 0, 0), (0, 2, 5, 1), (0, 1, 6, 1), (0, 2, 6, 1), (1, 1, 2, 1), (0, 9, 6, 1), (0, 9, 6, 0)]
    device, stream, count, want = zip(*asks)
    n = len(asks)
    out = (C.c_int * n)()
    host.b2h_wait_reports(n, (C.c_int * n)(*device), (C.c_ulonglong * n)(*stream), (C.c_uint * n)(*count), out)
    assert list(out) == list(want)


@pytest.fixture(scope="module")
def late(native, tmp_path_factory):
    pytest.importorskip("torch")
    so = str(tmp_path_factory.mktemp("late") / "liblate_tile.so")
    csrc = os.path.dirname(native.LIB)
    subprocess.run([native.NVCC] + native.NVCC_FLAGS + ["-shared", "-o", so, os.path.join(HERE, "fake", "late_tile.cu"), "-L", csrc, "-lb200mlp",
                                                       "-Xlinker", "-rpath=" + csrc], check=True)
    lib = C.CDLL(so)
    lib.late_launch.argtypes = [C.c_int, C.c_int] + [C.c_void_p] * 4
    lib.late_report.argtypes = [C.c_void_p, C.POINTER(C.c_uint), C.POINTER(C.c_int)]
    return lib


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0, 1, 2, 3])
def test_a_wait_that_runs_out(late, form):
    """Two streams' callers are both told, the kernels end within the bound, and the next ones run."""
    import torch
    ones, zeros = torch.ones(256, 128, device="cuda", dtype=torch.float16), torch.zeros(256, 128, device="cuda", dtype=torch.float16)
    out = torch.zeros(256, 256, device="cuda")
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def launch(late_):
        assert late.late_launch(form, late_, ones.data_ptr(), zeros.data_ptr(), out.data_ptr(), a.cuda_stream) == 0

    def report(s):
        count, news = C.c_uint(), C.c_int()
        assert late.late_report(s.cuda_stream, C.byref(count), C.byref(news)) == 0
        return count.value, news.value

    before = report(a)[0]
    report(b)
    assert report(a)[1] == 0 and report(b)[1] == 0
    t0 = time.time()
    launch(1)
    count, news = report(a)
    assert news == 1 and count > before and time.time() - t0 < 8.0
    assert report(b) == (count, 1)
    assert report(a) == (count, 0) and report(b) == (count, 0)
    launch(0)
    assert report(a) == (count, 0) and report(b) == (count, 0)
    assert bool((out == 128.0).all())


@pytest.mark.gpu
def test_sync_on_several_streams(native):
    torch = pytest.importorskip("torch")
    from tbb_test_b200 import lm
    h, w, t = torch.randn(40, 64, device="cuda"), torch.randn(90, 64, device="cuda"), torch.zeros(40, dtype=torch.int64, device="cuda")
    want = lm.xent(h, w, t)[0]
    for s in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            got = lm.xent(h, w, t)[0]
            lm.sync()
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_sync_takes_a_device_in_any_form(native):
    torch = pytest.importorskip("torch")
    from tbb_test_b200 import lm
    for device in (None, "cuda", "cuda:0", 0, torch.device("cuda"), torch.device("cuda", 0)):
        lm.sync(device)


def test_sync_refuses_other_devices(native):
    torch = pytest.importorskip("torch")
    from tbb_test_b200 import lm
    for device in ("cpu", torch.device("cpu")):
        with pytest.raises(ValueError):
            lm.sync(device)
