"""The C++ side of norm, clip and sample (tbb_test_b200/native) without a GPU: it loads, and refuses before any device work."""
import math

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
