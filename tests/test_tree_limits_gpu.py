"""The drafted-tree operators at the ends of what their arguments can say: sizes whose bytes pass 64
bits are refused before a launch, and counts beyond one launch's grid are more launches."""
import numpy as np
import pytest

from tests import tree_ref
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


# Rotations: 5 e (|l| + |r|) with e = 2^-24, as in tests/test_tree_gpu.py, 8 e allowed.
ROPE_E = 8 * 2.0 ** -24


@pytest.mark.parametrize("adjacent", [False, True])
def test_rope_at_of_more_tokens_than_a_launch_takes(gpu, up, adjacent):
    """2^24 + 5 tokens of one pair: 256 threads a token pass 2^32."""
    rng = np.random.default_rng(1)
    n = 2 ** 24 + 5
    x = rng.standard_normal((n, 2), dtype=np.float32)
    pos = rng.integers(0, 100000, n, dtype=np.int32)
    xb, pb = up(x), up(pos)
    gpu.rope_at(xb, pb, 1, 2, 1e4, 0.5, 2, n, adjacent=adjacent)
    got = np.frombuffer(gpu.read(xb, x.nbytes), np.float32).reshape(x.shape)
    bad = 0
    for i in range(0, n, 1 << 20):
        l, r = x[i:i + (1 << 20)].astype(np.float64).T
        a = pos[i:i + (1 << 20)] * 0.5
        want = np.stack([l * np.cos(a) - r * np.sin(a), l * np.sin(a) + r * np.cos(a)], 1)
        bad += int((np.abs(got[i:i + (1 << 20)] - want) > ROPE_E * (np.abs(l) + np.abs(r))[:, None]).sum())
    assert bad == 0


def test_rope_at_where_one_launch_of_whole_loads_follows_another(gpu, up):
    rng = np.random.default_rng(2)
    n, first = 2 ** 23 + 3, 2 ** 23 - 5
    x = np.zeros((n, 8), np.float32)
    x[:8], x[first:] = (rng.standard_normal((8, 8)) for _ in range(2))
    pos = rng.integers(0, 100000, n, dtype=np.int32)
    xb, pb = up(x), up(pos)
    gpu.rope_at(xb, pb, 1, 8, 1e4, 1.0, 8, n)
    for at in (0, first):
        got = np.frombuffer(gpu.read(xb, 8 * 32, at * 32), np.float32).reshape(8, 1, 8)
        old = x[at:at + 8].reshape(8, 1, 8).astype(np.float64)
        size = np.abs(old[..., :4]) + np.abs(old[..., 4:])
        assert np.all(np.abs(got - tree_ref.rope(old, pos[at:at + 8], 1e4, 1.0, 8, False)) <= ROPE_E * np.concatenate([size, size], -1)), at


def test_rope_at_of_more_heads_than_a_launch_takes(gpu, up):
    """65535 workgroups of 16 heads, and three heads more."""
    rng = np.random.default_rng(3)
    heads = 65535 * 16 + 3
    x = rng.standard_normal((2, heads, 2)).astype(np.float32)
    pos = np.array([7, 1234], np.int32)
    xb, pb = up(x), up(pos)
    gpu.rope_at(xb, pb, heads, 2, 1e4, 1.0, 2, 2)
    got = np.frombuffer(gpu.read(xb, x.nbytes), np.float32).reshape(x.shape)
    size = np.abs(x.astype(np.float64)).sum(-1, keepdims=True)
    assert np.all(np.abs(got - tree_ref.rope(x, pos, 1e4, 1.0, 2, False)) <= ROPE_E * size)


@pytest.mark.parametrize("nodes,heads,kv_heads", [(256, 4096, 1), (256, 2 ** 18, 2 ** 18), (1, 2 ** 21, 2 ** 21)])
def test_attention_tree_refuses_more_rows_than_a_launch_takes(gpu, nodes, heads, kv_heads):
    """65536 workgroups along y; 2^26 rows to join; more heads than the operator takes. Buffers of the whole size."""
    sizes = [4 * nodes * heads, 4 * nodes * kv_heads, 4 * nodes * kv_heads, 4 * nodes * heads, 4 * nodes]
    held = [gpu.buffer(n) for n in sizes]
    try:
        for op in (gpu.attention_tree, gpu.attention_tree_f16kv):
            refused(lambda: op(*held, heads, kv_heads, 1, 0, 1.0, 1 << 30, nodes, nodes), "more than a launch takes")
    finally:
        for b in held:
            gpu.destroy(b)


def test_attention_tree_of_the_most_rows_of_a_kv_head(gpu, up):
    """65535 workgroups along y, for one node: zero queries weigh its one key alone."""
    heads, hd = 65535 * 16, 1
    q, k, v, y = up(np.zeros(heads, np.float32)), up(np.zeros(1, np.float32)), up(np.full(1, 2.5, np.float32)), up(np.zeros(heads, np.float32))
    refused(lambda: gpu.attention_tree(q, k, v, y, up(np.array([-1], np.int32)), 2 ** 20 + 1, 1, hd, 0, 1.0, 9, 1, 1), "more than a launch takes")
    gpu.attention_tree(q, k, v, y, up(np.array([-1], np.int32)), heads, 1, hd, 0, 1.0, 9, 1, 1)
    assert np.all(np.frombuffer(gpu.read(y, 4 * heads), np.float32) == 2.5)
