"""What the token-model operators do before any GPU is involved: the refusal of sizes, the launch they would get, and
the definitions the GPU tests compare with (gradients against differences)."""
import ctypes as C

import numpy as np
import pytest

import token_reference as ref
from zigneuron_b200 import Backend, _lib

SHAPE, INVALID, NOT_INIT = 7, 1, 3
BIG = 1 << 31


def plan(op, a, b, c, sms=148):
    out = (C.c_int64 * 5)()
    status = _lib.lib.zn_debug_token_plan(op, a, b, c, sms, out)
    return status, dict(zip(("blocks", "threads", "share", "smem", "scratch"), out))


@pytest.mark.parametrize("op,a,b,c,status", [
    (0, 4, 0, 8, SHAPE), (0, 4, 8, 0, SHAPE), (0, BIG, 8, 8, SHAPE), (0, 4, BIG - 1, BIG - 1, SHAPE),
    (1, 4, 0, 8, SHAPE), (1, 4, 8, 0, SHAPE), (1, BIG - 1, 8, BIG - 1, SHAPE),
    (2, 4, 0, 0, SHAPE), (2, 4, 100, 129, INVALID), (2, BIG, 100, 0, SHAPE),
    (2, 1, (1 << 30) + 1, 0, SHAPE), (3, 1, (1 << 30) + 1, 0, SHAPE), (4, 1, (1 << 30) + 1, 1, SHAPE),
    (3, 4, 0, 0, SHAPE), (4, 4, 0, 1, SHAPE), (4, 4, 100, 0, SHAPE), (4, 4, 100, 513, SHAPE),
    (5, 0, 8, 32, SHAPE), (5, 8, 0, 32, SHAPE), (5, 8, 8, 48, INVALID), (5, 8, 8, 0, INVALID),
    (6, 1, 0, 8, SHAPE), (6, 1, 8, 0, SHAPE), (6, 1, BIG, 8, SHAPE), (7, 1, 1, 1, INVALID), (-1, 1, 1, 1, INVALID),
])
def test_sizes_that_are_refused(op, a, b, c, status):
    assert plan(op, a, b, c)[0] == status


def test_plan_arguments():
    assert _lib.lib.zn_debug_token_plan(0, 1, 1, 1, 148, None) == INVALID
    assert plan(0, 1, 1, 1, sms=0)[0] == INVALID


@pytest.mark.parametrize("op,c_values", [(0, (1, 7, 4096)), (1, (1, 7, 4096)), (2, (0, 1, 128)), (3, (0,)), (4, (1, 64, 512)), (5, (32, 128)), (6, (1, 129, 8192))])
def test_every_accepted_size_gets_a_launch_within_the_limits(op, c_values):
    for a in (1, 2, 31, 149, 4097, 1_000_000):
        for b in (1, 3, 1000, 50_001, 131_072, 1_000_003):
            for c in c_values:
                status, p = plan(op, a, b, c)
                assert status == 0, (op, a, b, c)
                assert 1 <= p["blocks"] < BIG and 32 <= p["threads"] <= 1024 and p["threads"] % 32 == 0
                assert p["share"] >= 1 and 0 <= p["smem"] <= 227 * 1024 and p["scratch"] >= 0


def test_null_context_is_refused():
    lib = _lib.lib
    assert lib.zn_embedding_forward(None, None, None, None, 1, 1, 1, 1.0) == NOT_INIT
    assert lib.zn_embedding_backward(None, None, None, None, 1, 1, 1, 1.0, 0) == NOT_INIT
    assert lib.zn_token_logprobs(None, None, 1, None, 1, 1, 1.0, 0, None, None, None, None, None) == NOT_INIT
    assert lib.zn_token_logprobs_backward(None, None, 1, None, None, None, None, None, None, 1, 1, 1, 1.0) == NOT_INIT
    assert lib.zn_distill_loss(None, None, 1, None, None, 1, 1, 1, 1.0, None, None, None, 1) == NOT_INIT
    assert lib.zn_quantize4(None, None, None, None, 1, 1, 32) == NOT_INIT
    assert lib.zn_matmul4_bias_act(None, None, None, None, None, None, 1, 1, 1, 32, 0) == NOT_INIT


def test_pointer_types_are_checked():
    with pytest.raises(TypeError):
        _lib.ptr(np.zeros(3, np.int64), np.int32)
    with pytest.raises(TypeError):
        _lib.ptr(np.zeros(3, np.int32))
    with pytest.raises(TypeError):
        _lib.ptr(np.zeros((4, 4), np.float32)[:, :2])


def test_packed_shapes():
    assert Backend.packed4_shape(10, 128, 64) == ((10, 16), (10, 2))
    assert Backend.packed4_shape(3, 129, 32) == ((3, 32), (3, 5))


def _difference(f, x, eps=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += eps
        down[i] -= eps
        g[i] = (f(up) - f(down)) / (2 * eps)
    return g


def test_reference_gradients_against_differences():
    """Central differences in float64: step 1e-5, so truncation near 1e-10 and rounding near 1e-11 of values of order 10."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 7)) * 2
    tok = np.array([4, -1, 0])
    gl, gh = rng.standard_normal(3), rng.standard_normal(3)
    for t in (0.5, 1.0, 2.0):
        def f(v):
            (lp, _), (h, _), _, _, _ = ref.token_logprobs(v, tok, t, 0)
            return (gl * lp).sum() + (gh * h).sum()
        assert np.allclose(ref.token_logprobs_backward(x, tok, t, gl, gh)[0], _difference(f, x), atol=1e-7)
        ids = np.array([[0, 3, 3], [-1, 6, 2], [-1, -1, -1]])
        u, w = rng.standard_normal((3, 3)), np.array([0.5, 2.0, 1.0])
        assert np.allclose(ref.distill_loss(x, ids, u, t, w)[1][0], _difference(lambda v: ref.distill_loss(v, ids, u, t, w)[0][0].sum(), x), atol=1e-7)


def test_reference_embedding_gradient_is_the_transpose_of_the_lookup():
    rng = np.random.default_rng(2)
    tok = np.array([3, 0, 3, -1, 1, 3])
    table, g = rng.standard_normal((5, 4)), rng.standard_normal((6, 4))
    grad = ref.embedding_backward(g, tok, 5, 0.5)[0]
    look = np.where(tok[:, None] >= 0, 0.5 * table[np.maximum(tok, 0)], 0)
    assert np.isclose((look * g).sum(), (table * grad).sum())


def test_packing_round_trip():
    """The layout in words: in each run of 16 words, word 4 i + t stands at place 4 t + i, the lowest code in the lowest bits."""
    codes = np.arange(2 * 256).reshape(2, 256) * 7 % 16
    words = ref.pack4(codes)
    for j in range(2):
        for i in range(256):
            w = i // 8
            place = w // 16 * 16 + (w % 4) * 4 + w % 16 // 4
            assert (int(words[j, place]) >> (4 * (i % 8))) & 15 == codes[j, i]
