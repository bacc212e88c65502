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
