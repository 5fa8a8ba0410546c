"""Engine.load_tensor_f8 against the model's own sizes: the C entry takes pointers and copies the whole tensor from them, so an array that is smaller, or has its
sides the other way round, must not reach it."""
import numpy as np
import pytest

from distributed_inference_server_b200 import Engine, ModelShape
from distributed_inference_server_b200 import binding as B

SHAPE = ModelShape(1024, 272, 2, 8, 2, 128, 1040, 512)
SIZES = {B.T_WQ: (1024, 272), B.T_WK: (256, 272), B.T_WV: (256, 272), B.T_WO: (272, 1024), B.T_WGATE: (1040, 272), B.T_WUP: (1040, 272), B.T_WDOWN: (272, 1040)}


class Recorded:
    def __init__(self):
        self.calls = []

    def dis_engine_load_tensor_f8(self, h, kind, layer, host, scale):
        self.calls.append((kind, layer))
        return B.OK


def engine():
    e = Engine.__new__(Engine)
    e.lib, e.h, e.shape = Recorded(), None, SHAPE
    return e


def pair(rows, cols):
    return np.zeros((rows, cols), np.uint8), np.zeros((-(-rows // 128), -(-cols // 128)), np.float32)


@pytest.mark.parametrize("kind", SIZES)
def test_whole_tensors_are_passed_on(kind):
    e = engine()
    e.load_tensor_f8(kind, 1, *pair(*SIZES[kind]))
    assert e.lib.calls == [(kind, 1)]


@pytest.mark.parametrize("kind", SIZES)
def test_other_sizes_are_refused(kind):
    rows, cols = SIZES[kind]
    for size in ((rows - 16, cols), (rows, cols - 16), (cols, rows), (rows // 2, cols), (rows, cols // 2), (rows + 128, cols), (16, 16)):
        e = engine()
        with pytest.raises(TypeError) as err:
            e.load_tensor_f8(kind, 0, *pair(*size))
        assert str(SIZES[kind][0]) in str(err.value) and e.lib.calls == []


def test_what_is_no_projection_is_left_to_the_engine():
    e = engine()
    for kind in (B.T_EMBED, B.T_ATTN_NORM, B.T_LM_HEAD, 77):
        e.load_tensor_f8(kind, 0, *pair(16, 16))  # (which refuses these before it reads anything)
    assert len(e.lib.calls) == 4
