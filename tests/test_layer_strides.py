"""The layer operators' checks of strides, without a GPU: the addresses are
never read, and a call that passes the checks fails at the device."""
import pytest

import lal_b200 as L
from lal_b200 import LalTailError
from test_layer_ops import A, ARG, D, E, F, norm, swiglu, weights

#: times four rows past 2^64 bytes, whatever the type
HUGE = [2 ** 62, 2 ** 62 + 8, 2 ** 63 - 1]


@pytest.mark.parametrize("stride", HUGE)
@pytest.mark.parametrize("call", [
    lambda n: norm(rows=5, x_stride=n), lambda n: norm(rows=5, q_stride=n), lambda n: norm(rows=5, d_h=F, h_stride=n),
    lambda n: norm(rows=5, d_h=F, d_residual=A + 0x100000, residual_stride=n),
    lambda n: swiglu(rows=5, gate_stride=n), lambda n: swiglu(rows=5, up_stride=n), lambda n: swiglu(rows=5, q_stride=n),
    lambda n: weights(rows=5).quantize(E, w_stride=n), lambda n: weights(rows=5).dequantize(E, w_stride=n),
    lambda n: weights().matvec(D, E, 5, F, y_stride=n), lambda n: weights().matvec(D, E, 5, F, xq_stride=n),
])
def test_rows_beyond_the_address_space_are_refused(call, stride):
    """The last row's offset in bytes passes 2^64: it may not wrap into a
    buffer that looks short."""
    with pytest.raises(LalTailError) as e:
        call(stride)
    assert e.value.code == ARG


def test_one_row_may_have_any_stride():
    for n in HUGE:
        with pytest.raises(LalTailError) as e:
            norm(rows=1, x_stride=n, q_stride=n)
        assert "stride" not in str(e.value)


# ---- columns of one buffer --------------------------------------------------------------------

#: rows of 1024 bytes: x in bytes 0-255, then the places named
@pytest.mark.parametrize("call", [
    lambda: norm(d_h=A + 256, x_stride=256, h_stride=256),
    lambda: norm(d_x=A + 512, d_h=A + 256, x_stride=256, h_stride=256),
    lambda: norm(d_x=A + 768, d_h=A, x_stride=256, h_stride=256),
    lambda: norm(d_q=A + 960, x_stride=256, q_stride=1024),
    lambda: norm(d_residual=A + 256, d_h=A + 512, d_q=A + 768, x_stride=256, residual_stride=256, h_stride=256, q_stride=1024),
    lambda: swiglu(d_up=A + 256, d_q=A + 512, gate_stride=256, up_stride=256, q_stride=1024),
    lambda: norm(d_scale=A + 256, x_stride=256),  # two scales between two rows
])
def test_columns_of_one_buffer_do_not_overlap(call):
    with pytest.raises(LalTailError) as e:
        call()
    assert "overlap" not in str(e.value)


@pytest.mark.parametrize("call", [
    lambda: norm(d_h=A + 252, x_stride=256, h_stride=256),              # the last value of x
    lambda: norm(d_x=A + 256, d_h=A + 4, x_stride=256, h_stride=256),   # the first
    lambda: norm(d_h=A + 772, x_stride=256, h_stride=256),              # h ends in the next row's x
    lambda: norm(d_h=A + 256, x_stride=256, h_stride=255),              # another step
    lambda: norm(d_q=A + 961, x_stride=256, q_stride=1024),
    lambda: norm(rows=200, d_scale=A + 256, x_stride=256),              # 200 scales reach the next row
    lambda: swiglu(d_up=A + 256, d_q=A + 448, gate_stride=256, up_stride=256, q_stride=1024),
])
def test_columns_that_overlap_are_refused(call):
    with pytest.raises(LalTailError) as e:
        call()
    assert e.value.code == ARG and "overlap" in str(e.value)
