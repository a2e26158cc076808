"""The C++ side of norm, clip and sample (tbb_test_b200/native) without a GPU: it loads, and refuses before any device work."""
import math
import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def test_it_is_built_in_tree_and_loads(native, lm):
    assert lm._native().__file__ == native.NATIVE


def test_what_is_no_tensor_of_a_gpu_is_refused(lm):
    x, v = torch.zeros(4, 8), torch.zeros(4)
    for call in (lambda: lm.norm(x), lambda: lm.norm(None), lambda: lm.norm([1.0]), lambda: lm.norm(v), lambda: lm.norm_e4m3(x), lambda: lm.norm_grad(x, x), lambda: lm.norm_grad(3, x),
                 lambda: lm.clip(x, 1.0), lambda: lm.clip([x, v], 1.0), lambda: lm.clip([], 1.0), lambda: lm.clip(5, 1.0), lambda: lm.clip([None], 1.0),
                 lambda: lm.clip(x, -1.0), lambda: lm.clip(x, math.nan), lambda: lm.clip(x, None, out=x), lambda: lm.clip([x], 1.0, out=[]), lambda: lm.sample(x, v),
                 lambda: lm.sample(x, 0.5), lambda: lm.sample(v, v)):
        with pytest.raises(ValueError):
            call()


def test_numbers_have_to_be_numbers(lm):
    x = torch.zeros(4, 8)
    for call in (lambda: lm._native().norm(x), lambda: lm._native().clip(x, 1.0, None, None), lambda: lm.clip([x], "much")):
        with pytest.raises(TypeError):
            call()


def test_an_8_bit_norm_without_a_block_is_refused(lm):
    """None is no number of columns, nor a norm in the type of x."""
    x = torch.zeros(4, 8)
    for block in (None, "128", 128.0):
        with pytest.raises(TypeError):
            lm.norm_e4m3(x, block=block)


def _torch_at(path, libraries=(), headers=()):
    """Where torch would lie, with these of its files."""
    for f in [path / "__init__.py", *[path / "lib" / f"lib{x}.so" for x in libraries], *[path / "include" / x for x in headers]]:
        f.parent.mkdir(parents=True, exist_ok=True)
        f.touch()
    return types.SimpleNamespace(origin=str(path / "__init__.py"))


@pytest.mark.parametrize("lacks", ["torch for CUDA", "torch's headers", "Python's headers", "CUDA's headers"])
def test_what_only_the_native_calls_need_stops_no_build(native, monkeypatch, tmp_path, capsys, lacks):
    """The C library and the driver need none of it: the build says what there is not, and ends as it should."""
    all_libraries = ["c10", "torch_cpu", "torch_python"] + ([] if lacks == "torch for CUDA" else ["c10_cuda", "torch_cuda"])
    spec = _torch_at(tmp_path / "torch", all_libraries, [] if lacks == "torch's headers" else ["torch/csrc/autograd/python_variable.h"])
    monkeypatch.setattr(native.importlib.util, "find_spec", lambda name: spec)
    monkeypatch.setattr(native, "NATIVE", str(tmp_path / "_lm_native.so"))
    paths = dict(native.sysconfig.get_paths())
    if lacks == "Python's headers":
        paths["include"] = str(tmp_path)
    monkeypatch.setattr(native.sysconfig, "get_paths", lambda: paths)
    if lacks == "CUDA's headers":
        monkeypatch.setattr(native, "NVCC", str(tmp_path / "bin" / "nvcc"))
    for call in (native.build_native, native.build_all):
        call()
        what = capsys.readouterr().err
        for name, file in (("torch for CUDA", "libc10_cuda.so"), ("torch for CUDA", "libtorch_cuda.so"), ("torch's headers", "python_variable.h"), ("Python's headers", "Python.h"),
                           ("CUDA's headers", "cuda_runtime_api.h")):
            assert (file in what) == (name == lacks)


@pytest.mark.parametrize("abi", [False, True])
def test_native_calls_are_built_with_torchs_own_abi(native, monkeypatch, tmp_path, abi):
    commands = []
    monkeypatch.setattr(native, "NATIVE", str(tmp_path / "_lm_native.so"))
    monkeypatch.setattr(native, "_run", lambda command, verbose: commands.append(command))
    monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: abi)
    assert native.build_native() == native.NATIVE
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(abi)}" in commands[0]
