"""The layer operators without a GPU: their refusals (arguments are checked
before any device call), calls that have nothing to do, and the 64-bit
definitions that the GPU tests hold the kernels to."""
import ctypes as C

import numpy as np
import pytest

import lal_b200 as L
import layer_ref as ref
from lal_b200 import LalTailError

ARG = 1
# addresses that no call dereferences: every one of these calls is refused or empty
A, B, D, E, F = (0x10000000 * i for i in range(1, 6))


def norm(**k):
    a = dict(d_x=A, d_residual=None, d_h=None, d_norm_w=B, eps=1e-6, rows=2, n_embd=64, d_q=D, d_scale=E)
    a.update(k)
    L.add_rms_norm_q8(**a)


@pytest.mark.parametrize("k", [
    dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(n_embd=0), dict(n_embd=-5), dict(n_embd=2 ** 30 + 1),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(d_x=None), dict(d_norm_w=None), dict(d_q=None), dict(d_scale=None),
    dict(d_residual=F),                        # a residual needs d_h
    dict(x_stride=63), dict(q_stride=63), dict(d_h=F, h_stride=63),
    dict(d_h=F, d_residual=A + 0x100000, residual_stride=63),
    dict(d_x=A + 2), dict(d_x=A + 1, dtype=L.LAL_TAIL_BF16), dict(d_norm_w=B + 2), dict(d_scale=E + 2),
    dict(d_q=A + 4 * 127),                     # q on the last value of x
    dict(d_h=A, h_stride=65),                  # h on x, with another stride
    dict(d_h=A + 4), dict(d_h=B), dict(d_scale=A), dict(d_scale=D + 100), dict(d_q=B),
])
def test_norm_refuses(k):
    with pytest.raises(LalTailError) as e:
        norm(**k)
    assert e.value.code == ARG and "add_rms_norm_q8" in str(e.value)


def swiglu(**k):
    a = dict(d_gate=A, d_up=B, rows=2, n=64, d_q=D, d_scale=E)
    a.update(k)
    L.swiglu_q8(**a)


@pytest.mark.parametrize("k", [
    dict(dtype=7), dict(rows=-1), dict(n=0), dict(n=2 ** 31 - 1), dict(d_gate=None), dict(d_up=None), dict(d_q=None),
    dict(d_scale=None), dict(gate_stride=63), dict(up_stride=1), dict(q_stride=0), dict(d_gate=A + 1),
    dict(d_up=B + 1, dtype=L.LAL_TAIL_F16), dict(d_scale=E + 1), dict(d_q=A), dict(d_scale=B), dict(d_q=E - 1),
])
def test_swiglu_refuses(k):
    with pytest.raises(LalTailError) as e:
        swiglu(**k)
    assert e.value.code == ARG and "swiglu_q8" in str(e.value)


def weights(d_q=A, d_scale=B, d_min=None, rows=4, cols=64, group=32):
    return L.Q4Weights(d_q, d_scale, d_min, rows, cols, group)


BAD_WEIGHTS = [dict(d_q=None), dict(d_scale=None), dict(d_q=A + 8), dict(d_scale=B + 1), dict(d_min=D + 1),
               dict(rows=-1), dict(cols=0), dict(cols=-32), dict(rows=2 ** 31 - 1), dict(cols=2 ** 31 - 1), dict(group=0), dict(group=16), dict(group=256)]


@pytest.mark.parametrize("k", BAD_WEIGHTS)
def test_bad_weights_are_refused_by_every_call(k):
    w = weights(**k)
    for call in (lambda: w.quantize(E), lambda: w.dequantize(E), lambda: w.matvec(E, F, 1, F + 0x1000)):
        with pytest.raises(LalTailError) as e:
            call()
        assert e.value.code == ARG


@pytest.mark.parametrize("name", ["quantize", "dequantize"])
@pytest.mark.parametrize("a,k", [((None,), {}), ((E,), dict(dtype=3)), ((E,), dict(w_stride=63)), ((E + 2,), {}),
                                 ((A,), {}), ((B,), {}), ((A - 4,), {})])
def test_quantizer_refuses(name, a, k):
    with pytest.raises(LalTailError) as e:
        getattr(weights(), name)(*a, **k)
    assert e.value.code == ARG


def test_quantizer_refuses_buffers_that_meet():
    with pytest.raises(LalTailError):
        weights(d_scale=A + 4 * 32 - 2).quantize(E)  # the scale begins inside the last row's blocks
    with pytest.raises(LalTailError):
        weights(d_min=B + 2).quantize(E)


@pytest.mark.parametrize("k", [
    dict(d_xq=None), dict(d_scale_x=None), dict(d_y=None), dict(n_streams=-1), dict(n_streams=257), dict(dtype=3),
    dict(xq_stride=63), dict(y_stride=3), dict(d_y=F + 2), dict(d_y=F + 1, dtype=L.LAL_TAIL_BF16),
    dict(d_scale_x=E + 2), dict(d_y=D), dict(d_y=E), dict(d_y=A), dict(d_y=B),
])
def test_matvec_refuses(k):
    a = dict(d_xq=D, d_scale_x=E, n_streams=2, d_y=F)
    a.update(k)
    with pytest.raises(LalTailError) as e:
        weights().matvec(**a)
    assert e.value.code == ARG and "q4_matvec" in str(e.value)


def test_nothing_to_do_needs_no_gpu():
    norm(rows=0)
    swiglu(rows=0)
    weights(rows=0).quantize(E)
    weights(rows=0).dequantize(E)
    weights(rows=0).matvec(D, E, 2, F)
    weights().matvec(D, E, 0, F)


def test_null_weights():
    assert L.lib().lal_tail_q4_matvec(None, D, 64, E, 1, F, 64, 0, None) == ARG


def test_description_mirrors_the_header():
    assert C.sizeof(L.Q4Desc) == 40
    assert L.Q4Weights.row_bytes(1) == 16 and L.Q4Weights.row_bytes(33) == 32
    assert L.Q4Weights.groups(129, 128) == 2


# ---- the definitions themselves ----------------------------------------------------------

def test_packing_is_a_round_trip():
    rng = np.random.default_rng(0)
    for cols in (1, 16, 31, 32, 33, 100):
        q = rng.integers(0, 16, (3, cols)).astype(np.uint8)
        p = ref.pack(q, fill=9)
        assert p.shape == (3, ref.row_bytes(cols))
        np.testing.assert_array_equal(ref.unpack(p, cols), q)
    # column 1 in byte 1's low half, column 17 in its high half
    q = np.zeros((1, 32), np.uint8)
    q[0, 1], q[0, 17] = 3, 5
    assert ref.pack(q)[0, 1] == 3 | 5 << 4


@pytest.mark.parametrize("minimum", [False, True])
def test_quantized_weights_are_half_a_step_off_at_most(minimum):
    rng = np.random.default_rng(1)
    w = (0.02 * rng.standard_normal((6, 200)) + 0.01).astype(np.float32).astype(np.float64)
    q, s, m = ref.quantize_q4(w, 64, minimum)
    back = ref.weights_q4(q, s, m, 64)
    step = s.astype(np.float64)[:, np.arange(200) // 64]
    assert np.all(np.abs(back - w) <= step / 2 * (1 + 1e-12))


def test_half_rounds_outwards():
    v = np.array([0.0, 1e-10, 1.0, 1.0001, 65504.0, 65505.0, 0.1])
    up, down = ref.half(v, True), ref.half(v, False)
    assert np.all(up.astype(np.float64) >= v) and np.all(down.astype(np.float64) <= v)
    assert up[1] == np.float16(2 ** -24) and np.isinf(up[5]) and up[2] == 1
