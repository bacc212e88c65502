"""The layer operators on the GPU (lal_tail_add_rms_norm_q8, lal_tail_swiglu_q8,
lal_tail_quantize_q4, lal_tail_dequantize_q4, lal_tail_q4_matvec) against their
definitions in 64 bits (layer_ref.py).

8-bit and 4-bit numbers and the f16 scales have to be equal: they are defined
as the roundings of 64-bit values.  Row scales are one rounding of a 64-bit
value to fp32, whose 64-bit sum and square root may differ in their last bits:
2^-24 relative, 2^-23 allowed.  A product's bound is derived at `bound`."""
import numpy as np
import pytest

import lal_b200 as L
import layer_ref as ref
import oracle
from lal_b200 import synth

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, L.LAL_TAIL_F32), "bf16": (torch.bfloat16, L.LAL_TAIL_BF16),
         "f16": (torch.float16, L.LAL_TAIL_F16)}
SENTINEL = 77


def stream():
    return torch.cuda.current_stream().cuda_stream


def padded(a, dtype, pad, behind=2):
    """Rows of `a` on the GPU, `pad` elements apart and with rows behind them,
    and the whole buffer."""
    rows, n = a.shape
    whole = torch.full((rows + behind, n + pad), SENTINEL, dtype=dtype, device="cuda")
    whole[:rows, :n] = torch.as_tensor(a).to(device="cuda", dtype=dtype)
    return whole[:rows, :n], whole


def untouched(whole, rows, n):
    return bool((whole[rows:] == SENTINEL).all()) and bool((whole[:rows, n:] == SENTINEL).all())


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def check_rows(q, scale, want_q, want_scale):
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    got, want = scale.cpu().numpy().astype(np.float64), want_scale.astype(np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    # 2^-23 relative, and the smallest step where the scale is subnormal
    assert np.all(np.abs(got[ok] - want[ok]) <= want[ok] * 2.0 ** -23 + 2.0 ** -149)


def activations(rng, rows, n):
    v = rng.standard_normal((rows, n))
    v[rng.random((rows, n)) < 0.005] *= 16.0
    return v


# ---- residual + RMSNorm ------------------------------------------------------------------

def run_norm(x, w, eps, dtype, r=None, pad=0, alias=None):
    t, code = TYPES[dtype]
    rows, n = x.shape
    dx, bx = padded(x, t, pad)
    dr, br = padded(r, t, pad + 1) if r is not None else (None, None)
    dw = torch.as_tensor(w, dtype=torch.float32).cuda()
    dh, bh = padded(np.zeros((rows, n)), t, pad + 2) if r is not None else (None, None)
    if alias == "x":
        dh, bh = dx, bx
    elif alias == "residual":
        dh, bh = dr, br
    dq, bq = padded(np.zeros((rows, n)), torch.int8, pad)
    ds, bs = padded(np.zeros((1, rows)), torch.float32, 3)
    h = dx.float() if r is None else (dx.float() + dr.float())
    want_h = h.to(t).clone()
    L.add_rms_norm_q8(dx.data_ptr(), dr.data_ptr() if r is not None else None,
                      dh.data_ptr() if dh is not None else None, dw.data_ptr(), eps, rows, n, dq.data_ptr(),
                      ds.data_ptr(), code, x_stride=n + pad, residual_stride=n + pad + 1,
                      h_stride=dh.stride(0) if dh is not None else None, q_stride=n + pad, stream=stream())
    torch.cuda.synchronize()
    if dh is not None:
        assert torch.equal(torch.nan_to_num(dh.float(), 5.0), torch.nan_to_num(want_h.float(), 5.0))
        assert untouched(bh, rows, n)
    assert untouched(bq, rows, n) and untouched(bs, 1, rows)
    return dq, ds[0], ref.norm_q8(f64(want_h), w.astype(np.float32), eps)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (2, 7), (1, 8), (3, 64), (33, 769), (4, 1024), (2, 3584), (5, 4096), (3, 4104),
                                    (2, 8192), (2, 18944), (1, 70001)])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_norm(dtype, rows, n, pad):
    rng = np.random.default_rng(rows * 1000 + n + pad)
    x, r = activations(rng, rows, n), activations(rng, rows, n)
    w = 1.0 + 0.2 * rng.standard_normal(n)
    for res in (None, r):
        q, s, want = run_norm(x, w, 1e-6, dtype, res, pad)
        check_rows(q, s, *want)


@pytest.mark.parametrize("alias", ["x", "residual"])
@pytest.mark.parametrize("n,pad", [(3584, 0), (100, 3)])
def test_norm_in_place(alias, n, pad):
    rng = np.random.default_rng(3)
    q, s, want = run_norm(activations(rng, 4, n), 1.0 + 0.1 * rng.standard_normal(n), 1e-5, "bf16",
                          activations(rng, 4, n), pad, alias)
    check_rows(q, s, *want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n", [15, 256, 1000])
def test_norm_rows_of_every_kind(dtype, n):
    """Zeros, one value, values that are not finite, the smallest and the
    largest numbers, and values halfway between two steps."""
    rng = np.random.default_rng(5)
    big = {"f32": 3e38, "bf16": 3e38, "f16": 6e4}[dtype]
    tiny = {"f32": 1e-40, "bf16": 1e-39, "f16": 6e-8}[dtype]
    x = rng.standard_normal((12, n))
    x[0] = 0.0
    x[1] = 0.0
    x[1, n // 2] = -3.0
    x[2, 0] = np.nan
    x[3, n - 1] = np.inf
    x[4, n // 3] = -np.inf
    x[5] = tiny * rng.integers(-9, 10, n)
    x[6] = big * rng.choice([-1.0, 1.0, 0.5], n)
    x[7] = 254.0 * rng.choice([-1.0, 1.0], n)
    x[7, 1:] = rng.integers(-253, 254, n - 1)  # 127 v / 254: half of them ties
    x[8] = 1e-3 * x[8]
    x[9] *= 1e-6 if dtype != "f16" else 1e-4
    x[10, 0] = big / 4  # all others round to 0
    q, s, want = run_norm(x, np.ones(n), 1e-6, dtype)
    check_rows(q, s, *want)
    assert np.isnan(s[2].item()) and np.isnan(s[3].item()) and s[0].item() == 0.0
    q, s, want = run_norm(x, 1.0 + 0.3 * rng.standard_normal(n), 0.0, dtype)  # eps 0
    check_rows(q, s, *want)


def test_norm_weights_of_every_kind():
    rng = np.random.default_rng(6)
    n = 300
    for w in (np.zeros(n), np.full(n, 1e30), np.full(n, 1e-30), np.where(np.arange(n) == 7, np.nan, 1.0),
              np.where(np.arange(n) == 9, np.inf, 1.0), np.full(n, -1.0)):
        q, s, want = run_norm(activations(rng, 3, n), w, 1e-6, "f32", activations(rng, 3, n))
        check_rows(q, s, *want)


# ---- SwiGLU ------------------------------------------------------------------------------

def run_swiglu(g, u, dtype, pad=0):
    t, code = TYPES[dtype]
    rows, n = g.shape
    both, _ = padded(np.concatenate([g, u], 1), t, pad)  # gate and up are columns of one buffer
    dg, du = both[:, :n], both[:, n:]
    dq, bq = padded(np.zeros((rows, n)), torch.int8, pad)
    ds, bs = padded(np.zeros((1, rows)), torch.float32, 3)
    L.swiglu_q8(dg.data_ptr(), du.data_ptr(), rows, n, dq.data_ptr(), ds.data_ptr(), code,
                gate_stride=both.stride(0), up_stride=both.stride(0), q_stride=n + pad, stream=stream())
    torch.cuda.synchronize()
    assert untouched(bq, rows, n) and untouched(bs, 1, rows)
    return dq, ds[0], ref.swiglu_q8(f64(dg), f64(du))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (2, 7), (1, 8), (33, 769), (4, 1024), (2, 3584), (3, 4104), (2, 18944),
                                    (1, 40001)])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_swiglu(dtype, rows, n, pad):
    rng = np.random.default_rng(rows * 1000 + n + pad)
    q, s, want = run_swiglu(activations(rng, rows, n), activations(rng, rows, n), dtype, pad)
    check_rows(q, s, *want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n", [16, 1000])
def test_swiglu_rows_of_every_kind(dtype, n):
    rng = np.random.default_rng(8)
    big = {"f32": 3e38, "bf16": 3e38, "f16": 6e4}[dtype]
    g, u = rng.standard_normal((14, n)), rng.standard_normal((14, n))
    g[0] = 0.0
    u[1] = 0.0
    g[2, 3] = np.nan
    u[3, n - 1] = np.nan
    g[4, 5] = np.inf
    g[5, 5] = -np.inf
    u[6, 0] = -np.inf
    g[7] = -rng.uniform(80.0, 110.0, n)    # exp(-gate) leaves 32 bits
    g[8] = -rng.uniform(300.0, 700.0, n)
    g[9] = rng.uniform(80.0, 700.0, n)
    g[10] = big
    u[10] = big * rng.choice([-1.0, 1.0], n)
    g[11] *= 1e-5
    u[11] *= 1e-5
    g[12, :] = -120.0
    g[12, 4] = 2.0                          # all others round to 0
    g[13] = -rng.uniform(800.0, 5000.0, n)  # exp(-gate) leaves 64 bits
    q, s, want = run_swiglu(g, u, dtype)
    check_rows(q, s, *want)


# ---- 4-bit weights -----------------------------------------------------------------------

class Weights:
    """Device buffers of [rows, cols] weights, from host numbers or empty."""

    def __init__(self, rows, cols, group, minimum, q=None, scale=None, low=None, fill=0):
        g = ref.row_bytes(cols), -(-cols // group)
        self.q = torch.full((rows + 1, g[0]), SENTINEL, dtype=torch.uint8, device="cuda")
        self.s = torch.full((rows + 1, g[1]), SENTINEL, dtype=torch.float16, device="cuda")
        self.m = torch.full((rows + 1, g[1]), SENTINEL, dtype=torch.float16, device="cuda") if minimum else None
        self.rows, self.cols = rows, cols
        if q is not None:
            self.q[:rows] = torch.as_tensor(ref.pack(q, fill)).cuda()
            self.s[:rows] = torch.as_tensor(scale).cuda()
            if minimum:
                self.m[:rows] = torch.as_tensor(low).cuda()
        self.w = L.Q4Weights(self.q.data_ptr(), self.s.data_ptr(), self.m.data_ptr() if minimum else None,
                             rows, cols, group)

    def untouched(self):
        return all(bool((t[self.rows:] == SENTINEL).all()) for t in (self.q, self.s, self.m) if t is not None)


def same(a, b):
    np.testing.assert_array_equal(a.astype(np.float64), b.astype(np.float64))  # NaN where NaN


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 31, 1), (2, 32, 0), (5, 33, 3), (4, 128, 0), (7, 200, 8),
                                           (9, 777, 0), (300, 1000, 5), (64, 3584, 0)])
def test_quantize_and_back(dtype, group, minimum, rows, cols, pad):
    rng = np.random.default_rng(cols + group)
    t, code = TYPES[dtype]
    dw, _ = padded(0.015 * rng.standard_normal((rows, cols)) + (0.003 if minimum else 0.0), t, pad)
    q, scale, low = ref.quantize_q4(f64(dw), group, minimum)
    w = Weights(rows, cols, group, minimum)
    w.w.quantize(dw.data_ptr(), code, w_stride=cols + pad, stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(ref.unpack(w.q[:rows].cpu().numpy(), cols), q)
    same(w.s[:rows].cpu().numpy(), scale)
    if minimum:
        same(w.m[:rows].cpu().numpy(), low)
    assert w.untouched()
    values = ref.weights_q4(q, scale, low, group)
    for out, (ot, ocode) in TYPES.items():
        back, whole = padded(np.zeros((rows, cols)), ot, pad)
        w.w.dequantize(back.data_ptr(), ocode, w_stride=cols + pad, stream=stream())
        torch.cuda.synchronize()
        assert untouched(whole, rows, cols)
        # in fp32 first (half a step of 2^-24 at most), then to the type
        np.testing.assert_array_equal(f64(back), f64(torch.as_tensor(values.astype(np.float32)).to(ot)))


@pytest.mark.parametrize("minimum", [False, True])
def test_quantize_groups_of_every_kind(minimum):
    """Zeros, one value, equal values, numbers that f16 scales cannot hold
    (too large: NaN; too small: rounded up to the smallest), borders."""
    rng = np.random.default_rng(4)
    w = rng.standard_normal((14, 96)).astype(np.float32)
    w[0] = 0.0
    w[1] = 0.0
    w[1, 40] = -2.5
    w[2] = 0.3
    w[3, 5] = np.nan
    w[4, 95] = np.inf
    w[5] *= 1e30
    w[6] *= 1e-9
    w[7] *= 1e-38
    w[8] = np.arange(96) % 29 - 14.0  # max 14: w / 2, half of them ties
    w[9] = rng.uniform(7e4, 9e4, 96)  # above f16, their spread is not
    w[10] = -w[9]
    w[11] = 1e-6 * rng.integers(-9, 9, 96)
    w[12] = 4.5e5 * rng.choice([-1.0, 1.0], 96)
    w[13] = np.arange(96) / 2.0
    q, scale, low = ref.quantize_q4(w.astype(np.float64), 32, minimum)
    dw = torch.as_tensor(w).cuda()
    d = Weights(14, 96, 32, minimum)
    d.w.quantize(dw.data_ptr(), L.LAL_TAIL_F32, stream=stream())
    torch.cuda.synchronize()
    same(d.s[:14].cpu().numpy(), scale)
    if minimum:
        same(d.m[:14].cpu().numpy(), low)
    np.testing.assert_array_equal(ref.unpack(d.q[:14].cpu().numpy(), 96), q)


# ---- product -----------------------------------------------------------------------------

def bound(y, size, cols, dtype):
    """What a result may be off.  A block's dot is exact and, scaled, rounded
    once (twice with a minimum); all blocks' terms are summed in 32 bits in
    some order, each partial sum at most `size`: (blocks + 10) 2^-24 of it.  The
    product with the stream's scale is rounded, and the result to its type."""
    eps = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    small = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dtype]
    return size * (cols / 32 + 11) * 2.0 ** -24 + np.abs(y) * (eps + 2.0 ** -23) + small


def vectors(rng, streams, cols):
    v = activations(rng, streams, cols)
    top = np.abs(v).max(1, keepdims=True)
    return np.rint(127 * v / top).astype(np.int8), (top[:, 0] / 127).astype(np.float32)


def random_weights(rng, rows, cols, group, minimum):
    groups = -(-cols // group)
    q = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    scale = (0.006 * (1 + 0.2 * rng.standard_normal((rows, groups)))).astype(np.float16)
    low = (scale * (-8 + 0.5 * rng.standard_normal((rows, groups)))).astype(np.float16) if minimum else None
    return q, scale, low


def run_matvec(xq, sx, d, dtype, pad=0):
    t, code = TYPES[dtype]
    streams = xq.shape[0]
    dx, _ = padded(xq, torch.int8, pad)
    ds = torch.as_tensor(sx).cuda()
    dy, whole = padded(np.zeros((streams, d.rows)), t, pad)
    d.w.matvec(dx.data_ptr(), ds.data_ptr(), streams, dy.data_ptr(), code, xq_stride=d.cols + pad,
               y_stride=d.rows + pad, stream=stream())
    torch.cuda.synchronize()
    assert untouched(whole, streams, d.rows)
    return dy


def check_matvec(rng, streams, rows, cols, group, minimum, dtype, pad):
    xq, sx = vectors(rng, streams, cols)
    q, scale, low = random_weights(rng, rows, cols, group, minimum)
    d = Weights(rows, cols, group, minimum, q, scale, low, fill=int(rng.integers(0, 16)))
    y = f64(run_matvec(xq, sx, d, dtype, pad))
    want, size = ref.matvec_q4(xq, sx, q, scale, low, group)
    off = np.abs(y - want) - bound(want, size, cols, dtype)
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("streams", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 48, 64, 65, 100, 128, 256])
def test_matvec_streams(streams, group, minimum):
    rng = np.random.default_rng(streams)
    check_matvec(rng, streams, 200, 640 + 32, group, minimum, "f32", 0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("streams", [1, 2, 7, 8, 20, 64])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (7, 31, 1), (16, 32, 0), (33, 100, 3), (129, 777, 0), (130, 1003, 5),
                                           (5, 4096, 0), (300, 128, 16), (64, 257, 8)])
def test_matvec_sizes(dtype, streams, rows, cols, pad):
    rng = np.random.default_rng(rows + cols)
    for group, minimum in ((32, True), (64, False), (128, True)):
        check_matvec(rng, streams, rows, cols, group, minimum, dtype, pad)


@pytest.mark.parametrize("streams", [1, 4, 13, 64])
@pytest.mark.parametrize("rows,cols", [(3584, 3584), (513, 18944), (5003, 896), (17, 50001)])
def test_matvec_large(streams, rows, cols):
    rng = np.random.default_rng(streams + cols)
    check_matvec(rng, streams, rows, cols, 128 if cols % 128 == 0 else 32, cols > 3584, "f32", 0)


@pytest.mark.parametrize("streams", [1, 3, 16, 70])
def test_matvec_values_of_every_kind(streams):
    """The extremes of 8 and 4 bits (xq -128 among them), a scale that is NaN
    in one row, a vector whose scale is NaN or 0: no other result is touched."""
    rng = np.random.default_rng(9)
    rows, cols = 70, 320
    for group, minimum in ((32, False), (128, True)):
        q, scale, low = random_weights(rng, rows, cols, group, minimum)
        xq = rng.choice(np.array([-128, 127], np.int8), (streams, cols))
        q[rng.random(q.shape) < 0.5] = 15
        sx = np.ones(streams, np.float32)
        xq[0, :] = -128
        scale[4, 1] = np.nan
        scale[7] = 0.0
        scale[8] = np.float16(6e-8)
        if streams > 2:
            sx[1], sx[2] = np.nan, 0.0
        d = Weights(rows, cols, group, minimum, q, scale, low, fill=15)
        y = f64(run_matvec(xq, sx, d, "f32"))
        with np.errstate(invalid="ignore"):
            want, size = ref.matvec_q4(xq, sx, q, scale, low, group)
        np.testing.assert_array_equal(np.isnan(y), np.isnan(want))
        ok = ~np.isnan(want)
        assert np.all((np.abs(y - want) <= bound(want, size, cols, "f32"))[ok])


def test_matvec_f16_overflows_to_infinity():
    q = np.full((3, 64), 15, np.uint8)
    d = Weights(3, 64, 64, False, q, np.full((3, 1), 100.0, np.float16))
    y = run_matvec(np.full((2, 64), 127, np.int8), np.ones(2, np.float32), d, "f16")
    assert bool(torch.isinf(y).all())


@pytest.mark.slow
def test_offsets_beyond_32_bits():
    rows, cols, group = 1_060_000, 4096, 128  # 2.17e9 bytes of 4-bit numbers
    q = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device="cuda")
    s = torch.full((rows, cols // group), 0.01, dtype=torch.float16, device="cuda")
    w = L.Q4Weights(q.data_ptr(), s.data_ptr(), None, rows, cols, group)
    rng = np.random.default_rng(2)
    for streams in (1, 9):
        xq, sx = vectors(rng, streams, cols)
        dx, ds = torch.as_tensor(xq).cuda(), torch.as_tensor(sx).cuda()
        y = torch.zeros(streams, rows, device="cuda")
        w.matvec(dx.data_ptr(), ds.data_ptr(), streams, y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        for at in (slice(0, 5), slice(rows - 5, rows)):
            qh, sh = ref.unpack(q[at].cpu().numpy(), cols), s[at].cpu().numpy()
            want, size = ref.matvec_q4(xq, sx, qh, sh, None, group)
            assert np.all(np.abs(f64(y[:, at]) - want) <= bound(want, size, cols, "f32"))
    del y
    # 4.3e9 values back, and to 4 bits again
    back = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    w.dequantize(back.data_ptr(), L.LAL_TAIL_BF16, stream=stream())
    last = back[-3:].clone()
    want = ref.weights_q4(ref.unpack(q[-3:].cpu().numpy(), cols), s[-3:].cpu().numpy(), None, group)
    np.testing.assert_array_equal(f64(last), f64(torch.as_tensor(want.astype(np.float32)).to(torch.bfloat16)))
    w.quantize(back.data_ptr(), L.LAL_TAIL_BF16, stream=stream())
    torch.cuda.synchronize()
    wq, ws, _ = ref.quantize_q4(f64(last), group, False)
    np.testing.assert_array_equal(ref.unpack(q[-3:].cpu().numpy(), cols), wq)
    same(s[-3:].cpu().numpy(), ws)
    # and 8-bit rows of them
    q8 = torch.empty(rows, cols, dtype=torch.int8, device="cuda")
    sc = torch.empty(rows, device="cuda")
    ones = torch.ones(cols, device="cuda")
    L.add_rms_norm_q8(back.data_ptr(), None, None, ones.data_ptr(), 1e-6, rows, cols, q8.data_ptr(), sc.data_ptr(),
                      L.LAL_TAIL_BF16, stream=stream())
    torch.cuda.synchronize()
    check_rows(q8[-3:], sc[-3:], *ref.norm_q8(f64(last), np.ones(cols, np.float32), 1e-6))
    half = cols // 2
    L.swiglu_q8(back.data_ptr(), back.data_ptr() + 2 * half, rows, half, q8.data_ptr(), sc.data_ptr(),
                L.LAL_TAIL_BF16, gate_stride=cols, up_stride=cols, q_stride=cols, stream=stream())
    torch.cuda.synchronize()
    check_rows(q8[-3:, :half], sc[-3:], *ref.swiglu_q8(f64(last)[:, :half], f64(last)[:, half:]))


# ---- refusals that need a GPU ------------------------------------------------------------

def test_host_memory_is_refused():
    x = torch.zeros(2, 64)
    d = torch.zeros(2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    q = torch.zeros(2, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(2, device="cuda")
    pinned = torch.zeros(2, 64).pin_memory()
    for bad in (x, pinned):
        with pytest.raises(L.LalTailError) as e:
            L.add_rms_norm_q8(bad.data_ptr(), None, None, w.data_ptr(), 1e-6, 2, 64, q.data_ptr(), s.data_ptr())
        assert e.value.code == 1 and "d_x" in str(e.value)
        with pytest.raises(L.LalTailError):
            L.swiglu_q8(d.data_ptr(), bad.data_ptr(), 2, 64, q.data_ptr(), s.data_ptr())
        with pytest.raises(L.LalTailError):
            L.Q4Weights(bad.data_ptr(), s.data_ptr(), None, 1, 64, 64).matvec(q.data_ptr(), s.data_ptr(), 1, d.data_ptr())
    # the refusals leave no error behind
    L.add_rms_norm_q8(d.data_ptr(), None, None, w.data_ptr(), 1e-6, 2, 64, q.data_ptr(), s.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert bool((s == 0).all())


# ---- a run of them together --------------------------------------------------------------

class Block:
    """One MLP block of a decode step and the tail behind it: norm, gate and
    up, SwiGLU, down, the residual, the tail's fused final norm."""

    def __init__(self, streams, d, f, group, dtype, seed=0):
        rng = np.random.default_rng(seed)
        self.t, self.code = TYPES[dtype]
        self.streams, self.d, self.f, self.dtype = streams, d, f, dtype
        self.gate_up = Weights(2 * f, d, group, False)
        self.down = Weights(d, f, group, True)
        for w, r, c in ((self.gate_up, 2 * f, d), (self.down, d, f)):
            full = torch.as_tensor(rng.standard_normal((r, c)) / np.sqrt(c), dtype=torch.float32).cuda()
            w.w.quantize(full.data_ptr(), L.LAL_TAIL_F32, stream=stream())
            torch.cuda.synchronize()
        self.norm_w = torch.as_tensor(1 + 0.1 * rng.standard_normal(d), dtype=torch.float32).cuda()
        e = lambda *s, **k: torch.empty(*s, device="cuda", **k)  # noqa: E731
        self.x, self.r, self.h, self.y = (e(streams, d, dtype=self.t) for _ in range(4))
        self.out = e(streams, d, dtype=torch.float32)
        self.gu = e(streams, 2 * f, dtype=self.t)
        self.q, self.aq = e(streams, d, dtype=torch.int8), e(streams, f, dtype=torch.int8)
        self.s, self.asc, self.s2 = e(streams), e(streams), e(streams)
        self.q2 = e(streams, d, dtype=torch.int8)

    def feed(self, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        for v in (self.x, self.r):
            v.copy_(torch.randn(self.streams, self.d, generator=g, device="cuda"))

    def run(self, st):
        n, d, f = self.streams, self.d, self.f
        L.add_rms_norm_q8(self.x.data_ptr(), self.r.data_ptr(), self.h.data_ptr(), self.norm_w.data_ptr(), 1e-6, n, d,
                          self.q.data_ptr(), self.s.data_ptr(), self.code, stream=st)
        self.gate_up.w.matvec(self.q.data_ptr(), self.s.data_ptr(), n, self.gu.data_ptr(), self.code, stream=st)
        L.swiglu_q8(self.gu.data_ptr(), self.gu.data_ptr() + f * self.gu.element_size(), n, f, self.aq.data_ptr(),
                    self.asc.data_ptr(), self.code, gate_stride=2 * f, up_stride=2 * f, stream=st)
        self.down.w.matvec(self.aq.data_ptr(), self.asc.data_ptr(), n, self.y.data_ptr(), self.code, stream=st)
        # the next norm adds the residual in place
        L.add_rms_norm_q8(self.y.data_ptr(), self.h.data_ptr(), self.h.data_ptr(), self.norm_w.data_ptr(), 1e-6, n, d,
                          self.q2.data_ptr(), self.s2.data_ptr(), self.code, stream=st)

    def outputs(self):
        return [t.clone() for t in (self.h, self.q, self.s, self.gu, self.aq, self.asc, self.y, self.q2, self.s2)]

    def check(self):
        """Every stage against its definition, on what the stage before it left."""
        first = (self.x.float() + self.r.float()).to(self.t)
        check_rows(self.q, self.s, *ref.norm_q8(f64(first), self.norm_w.cpu().numpy(), 1e-6))
        self.check_product(self.gate_up, self.q, self.s, self.gu, self.dtype)
        gu = f64(self.gu)
        check_rows(self.aq, self.asc, *ref.swiglu_q8(gu[:, :self.f], gu[:, self.f:]))
        self.check_product(self.down, self.aq, self.asc, self.y, self.dtype)
        last = (self.y.float() + first.float()).to(self.t)
        assert torch.equal(last, self.h)
        check_rows(self.q2, self.s2, *ref.norm_q8(f64(last), self.norm_w.cpu().numpy(), 1e-6))

    def check_product(self, w, q, s, y, dtype):
        low = w.m[:w.rows].cpu().numpy() if w.m is not None else None
        want, size = ref.matvec_q4(q.cpu().numpy(), s.cpu().numpy(), ref.unpack(w.q[:w.rows].cpu().numpy(), w.cols),
                                   w.s[:w.rows].cpu().numpy(), low, w.w.desc.group)
        assert np.all(np.abs(f64(y) - want) <= bound(want, size, w.cols, dtype))


@pytest.mark.parametrize("streams,dtype", [(1, "bf16"), (3, "f32"), (16, "f16"), (64, "bf16")])
def test_block(streams, dtype):
    b = Block(streams, 896, 1001, 32, dtype)
    for seed in (1, 2):
        b.feed(seed)
        b.run(stream())
        torch.cuda.synchronize()
        b.check()


@pytest.mark.parametrize("streams", [1, 8, 64])
def test_block_captured_and_replayed(streams):
    """Two graphs of two blocks, replayed in turn on one stream and at once on
    two, give what plain calls give: the calls share no workspace."""
    blocks = [Block(streams, 1024, 1536, 64, "bf16", seed=k) for k in range(2)]
    want = []
    for k, b in enumerate(blocks):
        b.feed(10 + k)
        b.run(stream())
        torch.cuda.synchronize()
        want.append(b.outputs())
    graphs = []
    for b in blocks:
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        b.feed(99)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            b.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    lanes = [torch.cuda.Stream() for _ in blocks]
    for at_once in (False, True):
        for k, b in enumerate(blocks):
            b.feed(10 + k)
        torch.cuda.synchronize()
        for _ in range(5):
            for k, g in enumerate(graphs):
                with torch.cuda.stream(lanes[k] if at_once else lanes[0]):
                    g.replay()
        torch.cuda.synchronize()
        for b, w in zip(blocks, want):
            for got, one in zip(b.outputs(), w):
                assert torch.equal(got, one)


def test_block_into_the_tail():
    """The block's sum is the residual stream that the tail's fused final norm
    takes: the token is the oracle's on the same values."""
    cfg = synth.CONFIGS["c1_gpt2"].with_(vocab=5003, n_embd=1024, hist=16)
    b = Block(1, 1024, 1536, 32, "f32")
    W = synth.lm_head_f32(cfg)
    rng = np.random.default_rng(1)
    w = (1.0 + 0.2 * rng.standard_normal(cfg.n_embd)).astype(np.float32)
    t = L.DecodeTail(cfg.vocab, cfg.n_embd, max_top_k=cfg.top_k, history_cap=cfg.hist)
    t.load_lm_head_f32(W)
    q, s = t.read_lm_head()
    hist = synth.history(cfg, 0)
    t.set_sampling([cfg.temperature], [cfg.top_k], [cfg.rep_penalty])
    t.set_history(0, hist)
    t.set_final_norm(w, 1e-6)
    port = oracle.PortLoop(q, s, hist, cfg.hist, cfg.temperature, cfg.top_k, cfg.rep_penalty, L.LAL_SAMPLER_LIBRARY)
    u, tok = torch.empty(1, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    for step in range(6):
        b.feed(step)
        draw = np.float32(rng.random())
        u.fill_(float(draw))
        torch.cuda.synchronize()
        b.run(t.stream())
        t.step_device(b.h.data_ptr(), 1, u.data_ptr(), tok.data_ptr())
        t.sync()
        want, _ = port.step(oracle.rms_norm(b.h[0].cpu().numpy(), w, 1e-6), draw)
        assert int(tok[0]) == want, step
    t.close()


def test_another_stream_and_thread():
    """Calls of two host threads on two streams at once."""
    import threading

    blocks = [Block(4, 512, 700, 32, "f16", seed=k) for k in range(2)]
    want = []
    for k, b in enumerate(blocks):
        b.feed(k)
        b.run(stream())
        torch.cuda.synchronize()
        want.append(b.outputs())
    failed = []

    def work(b):
        try:
            st = torch.cuda.Stream()
            for _ in range(50):
                b.run(st.cuda_stream)
            st.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(b,)) for b in blocks]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed
    for b, w in zip(blocks, want):
        for got, one in zip(b.outputs(), w):
            assert torch.equal(got, one)


FIRST_CALLS_IN_A_CAPTURE = """
import sys
sys.path[:0] = [%r, %r]
import torch
from test_gpu_layer_ops import Block

b = Block(%d, 1024, 1536, 64, "bf16")  # (its weights are quantized before)
b.feed(3)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b.run(torch.cuda.current_stream().cuda_stream)
g.replay()
torch.cuda.synchronize()
b.check()
print("captured")
"""


@pytest.mark.parametrize("streams", [1, 12, 40])
def test_first_calls_of_a_process_in_a_capture(streams):
    import os
    import subprocess
    import sys

    tests = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALLS_IN_A_CAPTURE % (os.path.dirname(tests), tests, streams)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_results_do_not_depend_on_other_streams_values():
    """A stream's results are the same bits whatever the other vectors hold,
    and in every run."""
    rng = np.random.default_rng(12)
    for streams in (2, 9, 20, 64, 70):
        q, scale, low = random_weights(rng, 300, 1000, 64, True)
        d = Weights(300, 1000, 64, True, q, scale, low)
        xq, sx = vectors(rng, streams, 1000)
        first = run_matvec(xq, sx, d, "f32")
        assert torch.equal(first, run_matvec(xq, sx, d, "f32"))
        other, so = vectors(rng, streams, 1000)
        other[1], so[1] = xq[1], sx[1]
        assert torch.equal(first[1], run_matvec(other, so, d, "f32")[1])


@pytest.mark.parametrize("streams,rows,cols", [(24, 40000, 1000), (32, 19001, 2100), (17, 152064, 260), (30, 12000, 3585),
                                               (16, 120000, 300), (8, 152064, 288), (48, 20000, 1500)])
def test_matvec_many_rows(streams, rows, cols):
    """More rows than a wave of tiles, ranges and tiles that end unevenly."""
    rng = np.random.default_rng(rows)
    check_matvec(rng, streams, rows, cols, 32, True, "bf16", 0)
    check_matvec(rng, streams, rows, cols, 128, False, "f32", 3)


@pytest.mark.parametrize("streams,cols", [(1, 1024), (3, 1003), (16, 1024), (20, 1003), (32, 1024), (64, 1024)])
def test_a_call_sees_what_the_call_before_it_wrote(streams, cols):
    """Calls follow each other with nothing between them, and each reads what
    the one before has just written over: sums in place, 8-bit rows, weights
    and their scales.  As when every call is waited for."""
    rows, rounds = 20000, 6
    rng = np.random.default_rng(3)
    w = Weights(rows, cols, 32, True)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    full = [torch.randn(rows, cols, generator=g, device="cuda") * (1 + k) for k in range(rounds)]
    r = [torch.randn(streams, cols, generator=g, device="cuda").to(torch.bfloat16) for _ in range(rounds)]
    norm_w = torch.as_tensor(1 + 0.1 * rng.standard_normal(cols), dtype=torch.float32).cuda()
    runs = []
    for wait in (True, False):
        h = torch.zeros(streams, cols, dtype=torch.bfloat16, device="cuda")
        q = torch.zeros(streams, cols, dtype=torch.int8, device="cuda")
        s = torch.zeros(streams, device="cuda")
        y = torch.zeros(rounds, streams, rows, device="cuda")
        torch.cuda.synchronize()
        for k in range(rounds):
            calls = [lambda k=k, j=j: L.add_rms_norm_q8(
                h.data_ptr(), r[(k + j) % rounds].data_ptr(), h.data_ptr(), norm_w.data_ptr(), 1e-6, streams, cols,
                q.data_ptr(), s.data_ptr(), L.LAL_TAIL_BF16, stream=stream()) for j in range(3)]
            calls.insert(1, lambda k=k: w.w.quantize(full[k].data_ptr(), stream=stream()))
            if k % 2:  # the norm, or the quantizer, directly before the product
                calls = calls[:1] + calls[2:] + calls[1:2]
            calls.append(lambda k=k: w.w.matvec(q.data_ptr(), s.data_ptr(), streams, y[k].data_ptr(), stream=stream()))
            for call in calls:
                call()
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        runs.append((h.clone(), q.clone(), s.clone(), y))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert all(bool((runs[0][3][k] != runs[0][3][k - 1]).any()) for k in range(1, rounds))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("streams", [2, 24, 64])
def test_products_on_two_streams_joined(streams, captured):
    """Gate and up at once on two streams behind one norm, joined at the
    SwiGLU; copies and a memset are what the operators follow and precede."""
    d, f = 1024, 2048
    x = activations(np.random.default_rng(1), streams, d)
    x_host = torch.as_tensor(x, dtype=torch.float32).pin_memory()
    weights = [Weights(f, d, 64, False) for _ in range(2)]
    for k, w in enumerate(weights):
        full = torch.randn(f, d, generator=torch.Generator().manual_seed(k)).cuda()
        w.w.quantize(full.data_ptr(), stream=stream())
        torch.cuda.synchronize()
    norm_w = torch.ones(d, device="cuda")
    dx, y = torch.empty(streams, d, device="cuda"), torch.empty(2, streams, f, device="cuda")
    q, aq = (torch.empty(streams, n, dtype=torch.int8, device="cuda") for n in (d, f))
    s, asc, out = torch.empty(streams, device="cuda"), torch.empty(streams, device="cuda"), torch.empty_like(aq)
    side, main = torch.cuda.Stream(), torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        dx.copy_(x_host, non_blocking=True)
        L.add_rms_norm_q8(dx.data_ptr(), None, None, norm_w.data_ptr(), 1e-6, streams, d, q.data_ptr(), s.data_ptr(),
                          stream=here.cuda_stream)
        side.wait_stream(here)
        weights[0].w.matvec(q.data_ptr(), s.data_ptr(), streams, y[0].data_ptr(), stream=here.cuda_stream)
        weights[1].w.matvec(q.data_ptr(), s.data_ptr(), streams, y[1].data_ptr(), stream=side.cuda_stream)
        here.wait_stream(side)
        L.swiglu_q8(y[0].data_ptr(), y[1].data_ptr(), streams, f, aq.data_ptr(), asc.data_ptr(), stream=here.cuda_stream)
        out.copy_(aq, non_blocking=True)
        y.zero_()

    with torch.cuda.stream(main):
        if captured:
            run()  # (a first run outside)
            torch.cuda.synchronize()
            out.zero_(), asc.zero_()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=main):
                run()
            for _ in range(4):
                graph.replay()
        else:
            for _ in range(4):
                run()
    torch.cuda.synchronize()
    # one call after another
    want = torch.empty_like(y)
    L.add_rms_norm_q8(dx.data_ptr(), None, None, norm_w.data_ptr(), 1e-6, streams, d, q.data_ptr(), s.data_ptr(), stream=stream())
    for k in range(2):
        weights[k].w.matvec(q.data_ptr(), s.data_ptr(), streams, want[k].data_ptr(), stream=stream())
        torch.cuda.synchronize()
    wq, ws = ref.swiglu_q8(f64(want[0]), f64(want[1]))
    check_rows(out, asc, wq, ws)
    assert bool((y == 0).all())


@pytest.mark.parametrize("streams", [12, 64])
def test_block_into_the_batched_tail_without_waiting(streams):
    """Blocks and batched steps one behind the other on the tail's stream give
    the tokens that they give when each is waited for."""
    cfg = synth.CONFIGS["c1_gpt2"].with_(vocab=5003, n_embd=1024, hist=16)
    b = Block(streams, 1024, 1536, 32, "f32")
    rng = np.random.default_rng(1)
    w = (1.0 + 0.2 * rng.standard_normal(cfg.n_embd)).astype(np.float32)
    u = torch.rand(8, streams, generator=torch.Generator().manual_seed(2)).cuda()
    tokens = []
    for wait in (True, False):
        t = L.DecodeTail(cfg.vocab, cfg.n_embd, max_top_k=cfg.top_k, history_cap=cfg.hist,
                         max_streams=streams)
        t.load_lm_head_f32(synth.lm_head_f32(cfg))
        t.set_sampling([cfg.temperature] * streams, [cfg.top_k] * streams, [cfg.rep_penalty] * streams)
        for k in range(streams):
            t.set_history(k, synth.history(cfg, k))
        t.set_final_norm(w, 1e-6)
        tok = torch.empty(8, streams, dtype=torch.int32, device="cuda")
        b.feed(4)
        torch.cuda.synchronize()
        for step in range(8):
            b.run(t.stream())
            t.step_device(b.h.data_ptr(), streams, u[step].data_ptr(), tok[step].data_ptr())
            if wait:
                t.sync()
        t.sync()
        tokens.append(tok.cpu())
        t.close()
    assert torch.equal(tokens[0], tokens[1])
    assert len(torch.unique(tokens[0])) > 1
