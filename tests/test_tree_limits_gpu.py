"""The drafted-tree operators at the ends of what their arguments can say: sizes whose bytes pass 64
bits are refused before a launch."""
import numpy as np
import pytest

from webgpu_amd.gpu import WgdError, WGD_E_INVALID

pytestmark = pytest.mark.gpu


@pytest.fixture
def up(gpu):
    held = []

    def upload(array):
        held.append(gpu.upload(np.ascontiguousarray(array)))
        return held[-1]

    yield upload
    for b in held:
        gpu.destroy(b)


def refused(call, about):
    with pytest.raises(WgdError) as e:
        call()
    assert e.value.status == WGD_E_INVALID and about in str(e.value), str(e.value)


def test_rope_at_refuses_rows_whose_bytes_pass_64_bits(gpu, up):
    """2^31 strides of 2^31 floats are 2^64 bytes: the rows do not fit, whatever the positions' buffer holds."""
    x, positions = up(np.zeros(64, np.float32)), up(np.zeros(64, np.int32))
    for offset in (0, 64):
        refused(lambda: gpu.rope_at(x, positions, 1, 2, 1e4, 1.0, 2, 2 ** 31 + 1, stride=2 ** 31, offset=offset), "rope_at input")
    refused(lambda: gpu.rope_at(x, positions, 1, 2, 1e4, 1.0, 2, 2 ** 32 - 1, stride=2 ** 32 - 1), "rope_at input")


def test_sample_rows_refuses_rows_whose_bytes_pass_64_bits(gpu, up):
    logits, uniforms, tokens = up(np.zeros(64, np.float32)), up(np.zeros(8, np.float64)), up(np.zeros(8, np.int32))
    refused(lambda: gpu.sample_rows(logits, 16, 2 ** 31 + 1, uniforms, tokens, 0.5, stride=2 ** 31), "sample_rows logits")
    refused(lambda: gpu.sample_rows(logits, 16, 2 ** 32 - 1, uniforms, tokens, 0.5, stride=2 ** 32 - 1), "sample_rows logits")
