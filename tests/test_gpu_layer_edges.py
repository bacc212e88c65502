"""The layer operators on the GPU where 32 bits, a kernel's shape or the order
of calls decide: what test_gpu_layer_ops.py does not reach.  Definitions and
tolerances are that file's."""
import numpy as np
import pytest


torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_layer_ops import check_rows, run_swiglu  # noqa: E402


# ---- SwiGLU at gates that 32-bit intermediates do not hold --------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,pad", [(8, 16, 0), (8, 1000, 3), (9, 4104, 0), (300, 1024, 0), (300, 4099, 1), (8, 70001, 0)])
def test_swiglu_extreme_gates(dtype, rows, n, pad):
    """Gates whose product with log2 e overflows, subnormal gates (halved they
    lose bits), gate * up that overflows where the result does not; with ups
    that put the row's largest value in the middle of fp32's range."""
    rng = np.random.default_rng(n)
    g, u = rng.standard_normal((rows, n)), rng.standard_normal((rows, n))
    g[0] = 2.4e38
    u[0] = 1e-10 * rng.uniform(0.1, 1.0, n)
    g[1, n // 2] = 3e38  # one of a row; the others round to 0
    u[1, n // 2] = -1e-3
    g[2] = rng.uniform(2.3e38, 3.3e38, n)
    u[2] = 1e-38 * rng.standard_normal(n)
    g[3] = 2.0 ** -133 * rng.integers(-60, 61, n)  # subnormal, and held by bf16
    u[3] = 1e38 * rng.uniform(-1.0, 1.0, n)
    g[4] = 2.0 ** -133 * rng.integers(1, 4, n)
    u[4] = 1e33
    g[5] = -rng.uniform(60.0, 79.0, n)
    u[5] = 1e38 * rng.uniform(-1.0, 1.0, n)  # gate * up overflows
    g[6] = rng.uniform(-1e-38, 1e-38, n)  # subnormal and the smallest normal ones
    u[6] = 1e30 * rng.standard_normal(n)
    g[7, 0] = 3e38
    u[7, 0] = 0.0
    if dtype == "f32":
        g[4, n // 3] = 3 * 2.0 ** -149
        u[4, n // 3] = 3e38
    q, s, want = run_swiglu(g, u, dtype, pad)
    assert np.isfinite(want[1]).all() and (want[1] > 0).all()
    check_rows(q, s, *want)
