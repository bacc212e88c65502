"""Every kernel of lal_tail_q4_matvec against the definition in 64 bits, at
shapes that reach it, which the kernels' names in a trace confirm.  The
definition is layer_ref.matvec_q4's, on the GPU (its sizes take numpy
minutes); the bound is test_gpu_layer_ops.bound."""
import numpy as np
import pytest

import layer_ref as ref
import lal_b200 as L

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_layer_ops import TYPES, bound, f64, stream  # noqa: E402

F64 = torch.float64


class Case:
    """Random weights and vectors on the GPU; `pad` columns behind each vector
    and each row of results."""

    def __init__(self, streams, rows, cols, group, minimum, seed=0, pad=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1000 * streams + cols)
        self.streams, self.rows, self.cols, self.group, self.pad = streams, rows, cols, group, pad
        groups = -(-cols // group)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.q = torch.randint(0, 256, (rows, ref.row_bytes(cols)), dtype=torch.uint8, generator=g, device="cuda")
        self.s = (0.006 * (1 + 0.2 * rand(rows, groups))).half()
        self.m = (self.s * (-8 + 0.5 * rand(rows, groups))).half() if minimum else None
        x = rand(streams, cols)
        x[torch.rand(streams, cols, generator=g, device="cuda") < 0.005] *= 16.0
        top = x.abs().amax(1, keepdim=True)
        self.x = torch.full((streams, cols + pad), 55, dtype=torch.int8, device="cuda")
        self.x[:, :cols] = torch.round(127 * x / top).to(torch.int8)
        self.sx = (top[:, 0] / 127).contiguous()
        self.w = L.Q4Weights(self.q.data_ptr(), self.s.data_ptr(), self.m.data_ptr() if minimum else None, rows, cols, group)

    def run(self, dtype="f32"):
        t, code = TYPES[dtype]
        whole = torch.full((self.streams + 1, self.rows + self.pad), 77, dtype=t, device="cuda")
        self.w.matvec(self.x.data_ptr(), self.sx.data_ptr(), self.streams, whole.data_ptr(), code,
                      xq_stride=self.cols + self.pad, y_stride=self.rows + self.pad, stream=stream())
        torch.cuda.synchronize()
        assert bool((whole[self.streams] == 77).all()) and bool((whole[:, self.rows:] == 77).all())
        return whole[:self.streams, :self.rows]

    def definition(self):
        """(y, the sum of its terms' sizes), as layer_ref.matvec_q4."""
        b = self.q.view(self.rows, -1, 16)
        n = torch.cat([b & 15, b >> 4], 2).view(self.rows, -1)[:, :self.cols]
        x = self.x[:, :self.cols].to(F64)
        y = torch.zeros(self.streams, self.rows, dtype=F64, device="cuda")
        size = torch.zeros_like(y)
        for c in range(0, self.cols, 32):
            k = slice(c, min(self.cols, c + 32))
            s = self.s[:, c // self.group].to(F64)
            if self.m is None:
                parts = [x[:, k] @ (n[:, k].to(F64) - 8.0).T * s]
            else:
                parts = [x[:, k] @ n[:, k].to(F64).T * s, x[:, k].sum(1)[:, None] * self.m[:, c // self.group].to(F64)]
            for p in parts:
                y += p
                size += p.abs()
        sx = self.sx.to(F64)[:, None]
        return y * sx, size * sx.abs()

    def check(self, y, dtype="f32"):
        want, size = (v.cpu().numpy() for v in self.definition())
        off = np.abs(f64(y) - want) - bound(want, size, self.cols, dtype)
        assert np.all(off <= 0), (float(off.max()), np.unravel_index(off.argmax(), off.shape))


def kernels_of(call):
    """The names of the kernels that `call` launches."""
    from torch.profiler import ProfilerActivity, profile

    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    return [e.name for e in p.events() if "q4_" in e.name]


def test_the_definition_on_the_gpu_is_the_other_one():
    for minimum in (False, True):
        c = Case(3, 40, 200, 64, minimum)
        q = ref.unpack(c.q.cpu().numpy(), c.cols)
        want, size = ref.matvec_q4(c.x.cpu().numpy(), c.sx.cpu().numpy(), q, c.s.cpu().numpy(),
                                   c.m.cpu().numpy() if minimum else None, 64)
        y, s = c.definition()
        np.testing.assert_allclose(f64(y), want, rtol=1e-12, atol=1e-12)
        np.testing.assert_allclose(f64(s), size, rtol=1e-12)


#: kernel -> shapes (streams, rows, columns, padding) for 148 SMs.  All begin rows at
#: 16-byte boundaries and fill whole stages of scales, but the last column block and the
#: last tile of rows end unevenly.
SHAPES = {
    "q4_wide_kernel": [(24, 40000, 1008, 0), (32, 19001, 2032, 16), (17, 152064, 512, 0), (29, 18944, 240, 0)],
    "q4_tc_kernel": [(48, 20000, 1520, 0), (64, 40001, 1008, 16), (33, 19001, 512, 0), (64, 3584, 4096, 0), (40, 1000, 2032, 0),
                     (64, 100, 18928, 0), (256, 20001, 240, 0), (63, 128, 256, 0)],
    "q4_mma_kernel<2, 2": [(16, 120000, 496, 0), (9, 113700, 1008, 0), (16, 5003, 1008, 16), (12, 513, 4080, 0), (24, 1000, 1008, 0)],
    "q4_mma_kernel<2, 1": [(8, 152064, 496, 0), (3, 113701, 240, 16), (8, 37888, 1264, 0), (5, 19007, 2048, 0)],
    "q4_mma_kernel<1, 1": [(1, 3584, 1008, 0), (7, 301, 496, 16), (4, 5000, 2032, 0), (8, 17, 18928, 0)],
}


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("minimum", [False, True])
@pytest.mark.parametrize("kernel,shape", [(k, s) for k, v in SHAPES.items() for s in v])
def test_matvec_kernel(kernel, shape, group, minimum):
    streams, rows, cols, pad = shape
    c = Case(streams, rows, cols, group, minimum, pad=pad)
    dtype = sorted(TYPES)[(streams + group // 32) % 3]
    c.check(c.run(dtype), dtype)


@pytest.mark.parametrize("kernel", sorted(SHAPES))
def test_the_shapes_reach_their_kernels(kernel):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the shapes are for 148 SMs")
    for streams, rows, cols, pad in SHAPES[kernel]:
        for group in (32, 64, 128):
            c = Case(streams, rows, cols, group, False, pad=pad)
            names = kernels_of(c.run)
            if not names:
                pytest.skip("no kernels in the trace")
            for name in names:
                # q4_mma_kernel<rows / 16, streams / 8, group, minima, fill>: never the fill of unaligned rows
                assert kernel in name and "MmaFill)2" not in name, (streams, rows, cols, group, name)


ONE_EACH = [(1, 3584, 1024), (8, 37888, 1280), (8, 120000, 256), (16, 5003, 1024), (16, 120000, 256), (24, 20000, 1024),
            (64, 20000, 1024), (64, 1000, 4096)]


@pytest.mark.parametrize("streams,rows,cols", ONE_EACH)
def test_aligned_results_do_not_depend_on_other_streams(streams, rows, cols):
    c = Case(streams, rows, cols, 64, True)
    first = c.run()
    assert torch.equal(first, c.run())
    if streams > 1:
        keep = c.x[1].clone(), c.sx[1].clone()
        c.x.copy_(c.x.flip(0))
        c.sx.copy_(2 * c.sx.flip(0))
        c.x[1], c.sx[1] = keep
        assert torch.equal(first[1], c.run()[1])


@pytest.mark.parametrize("group,minimum", [(32, False), (128, True)])
@pytest.mark.parametrize("streams,rows,cols", ONE_EACH)
def test_aligned_values_of_every_kind(streams, rows, cols, group, minimum):
    """The extremes of 8 and 4 bits, scales that are NaN, 0 or subnormal in one
    row, vectors' scales that are NaN or 0."""
    c = Case(streams, rows, cols, group, minimum)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    c.x.copy_(torch.where(torch.rand(c.x.shape, generator=g, device="cuda") < 0.5, -128, 127))
    c.x[0] = -128
    c.q[torch.rand(c.q.shape, generator=g, device="cuda") < 0.5] = 255
    c.sx.fill_(1.0)
    c.s[4, 1] = float("nan")
    c.s[7] = 0.0
    c.s[8] = 6e-8
    if streams > 2:
        c.sx[1], c.sx[2] = float("nan"), 0.0
    y = c.run()
    want, size = (v.cpu().numpy() for v in c.definition())
    got = f64(y)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(got - want) <= bound(want, size, cols, "f32"))[ok])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("streams,rows,cols", ONE_EACH + [(5, 300, 1000), (20, 300, 1000)])
def test_minima_far_below_their_scales(streams, rows, cols, group):
    """Groups of one large weight and many small ones, as an outlier makes
    them: where q is 0 the weight is the minimum alone, and no term of the
    scale's size enters the sum."""
    c = Case(streams, rows, cols, group, True)
    c.s.copy_((c.s.float() * 1e4).half())
    c.m.copy_((c.m.float() * 1e-2).half())
    c.q.zero_()
    c.x[:, ::group] = 0
    c.q[:, ::group // 2] |= 15  # the first column of each group, and x there is 0
    c.check(c.run())
    c.x[:, group // 2::group] = 0
    c.q[:, :16] = 0x21  # a block of small q's among them
    c.check(c.run())
