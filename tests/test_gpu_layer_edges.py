"""The layer operators on the GPU where 32 bits, a kernel's shape or the order
of calls decide: what test_gpu_layer_ops.py does not reach.  Definitions and
tolerances are that file's."""
import numpy as np
import pytest

import lal_b200 as L
import layer_ref as ref
from lal_b200 import synth

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_layer_ops import Weights, check_rows, f64, run_swiglu, stream  # noqa: E402


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


# ---- the chain into the one-stream tail ---------------------------------------------------

class MixedBlock:
    """An MLP block whose residual stream is fp32, as the tail's hidden vectors
    are, and whose gate and up are bf16; h and y run on from step to step."""

    def __init__(self, streams, d, f, group, seed=0):
        rng = np.random.default_rng(seed)
        self.n, self.d, self.f = streams, d, f
        self.gate_up, self.down = Weights(2 * f, d, group, False), Weights(d, f, group, True)
        for w, r, c in ((self.gate_up, 2 * f, d), (self.down, d, f)):
            full = torch.as_tensor(rng.standard_normal((r, c)) / np.sqrt(c), dtype=torch.float32).cuda()
            w.w.quantize(full.data_ptr(), L.LAL_TAIL_F32, stream=stream())
            torch.cuda.synchronize()
        self.norm_w = torch.as_tensor(1 + 0.1 * rng.standard_normal(d), dtype=torch.float32).cuda()
        self.start = torch.as_tensor(rng.standard_normal((2, streams, d)), dtype=torch.float32).cuda()
        self.h, self.y = torch.empty_like(self.start[0]), torch.empty_like(self.start[0])
        self.gu = torch.empty(streams, 2 * f, dtype=torch.bfloat16, device="cuda")
        self.q, self.aq = (torch.empty(streams, k, dtype=torch.int8, device="cuda") for k in (d, f))
        self.s, self.asc = (torch.empty(streams, device="cuda") for _ in range(2))

    def reset(self):
        self.h.copy_(self.start[0])
        self.y.copy_(self.start[1])

    def calls(self, st):
        n, d, f = self.n, self.d, self.f
        return [
            lambda: L.add_rms_norm_q8(self.y.data_ptr(), self.h.data_ptr(), self.h.data_ptr(), self.norm_w.data_ptr(), 1e-6,
                                      n, d, self.q.data_ptr(), self.s.data_ptr(), L.LAL_TAIL_F32, stream=st),
            lambda: self.gate_up.w.matvec(self.q.data_ptr(), self.s.data_ptr(), n, self.gu.data_ptr(), L.LAL_TAIL_BF16, stream=st),
            lambda: L.swiglu_q8(self.gu.data_ptr(), self.gu.data_ptr() + 2 * f, n, f, self.aq.data_ptr(), self.asc.data_ptr(),
                                L.LAL_TAIL_BF16, gate_stride=2 * f, up_stride=2 * f, stream=st),
            lambda: self.down.w.matvec(self.aq.data_ptr(), self.asc.data_ptr(), n, self.y.data_ptr(), L.LAL_TAIL_F32, stream=st),
            # the sum that the tail takes, directly before its step
            lambda: L.add_rms_norm_q8(self.y.data_ptr(), self.h.data_ptr(), self.h.data_ptr(), self.norm_w.data_ptr(), 1e-6,
                                      n, d, self.q.data_ptr(), self.s.data_ptr(), L.LAL_TAIL_F32, stream=st),
        ]


@pytest.mark.parametrize("streams,sampler,per_stream", [(1, L.LAL_SAMPLER_LIBRARY, False), (1, L.LAL_SAMPLER_SERVER, False),
                                                        (3, L.LAL_SAMPLER_LIBRARY, True), (5, L.LAL_SAMPLER_LIBRARY, False),
                                                        (1, L.LAL_SAMPLER_GPT2, False)])
def test_chain_into_the_tail_without_waiting(monkeypatch, streams, sampler, per_stream):
    """The tail starts while the norm before it ends, and takes the h that this
    norm writes: the tokens are those of a run that waits after every call."""
    if per_stream:
        monkeypatch.setenv("LAL_TAIL_PER_STREAM", "1")
    cfg = synth.CONFIGS["c1_gpt2"].with_(vocab=5003, n_embd=1024, hist=16)
    b = MixedBlock(streams, 1024, 1536, 32)
    w = (1.0 + 0.2 * np.random.default_rng(1).standard_normal(cfg.n_embd)).astype(np.float32)
    head = synth.lm_head_f32(cfg)
    steps = 24
    u = torch.rand(steps, streams, generator=torch.Generator().manual_seed(2)).cuda()
    runs = []
    for wait in (True, False):
        t = L.DecodeTail(cfg.vocab, cfg.n_embd, max_top_k=cfg.top_k, history_cap=cfg.hist, max_streams=streams, sampler=sampler)
        t.load_lm_head_f32(head)
        t.set_sampling([cfg.temperature] * streams, [cfg.top_k] * streams, [cfg.rep_penalty] * streams)
        for k in range(streams):
            t.set_history(k, synth.history(cfg, k))
        if sampler != L.LAL_SAMPLER_GPT2:
            t.set_final_norm(w, 1e-6)
        tok = torch.empty(steps, streams, dtype=torch.int32, device="cuda")
        b.reset()
        torch.cuda.synchronize()
        calls = b.calls(t.stream())
        for step in range(steps):
            for call in calls + [lambda: t.step_device(b.h.data_ptr(), streams, u[step].data_ptr(), tok[step].data_ptr())]:
                call()
                if wait:
                    t.sync()
        t.sync()
        torch.cuda.synchronize()
        runs.append((tok.cpu(), b.h.clone(), b.y.clone()))
        t.close()
    for one, two in zip(*runs):
        assert torch.equal(one, two)
    assert len(torch.unique(runs[0][0])) > 1


# ---- columns of one buffer ----------------------------------------------------------------

@pytest.mark.parametrize("rows,n", [(3, 64), (5, 1001), (301, 256)])
def test_operators_within_one_buffer(rows, n):
    """Rows of one record each: x, residual, h and q of the norm, gate, up and
    q of the SwiGLU, side by side."""
    rng = np.random.default_rng(n)
    x, r = rng.standard_normal((2, rows, n))
    w = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    step = 4 * n + 4  # in fp32: x, residual, h, q (in n / 4 of them) and a gap
    whole = torch.full((rows, step), 77.0, device="cuda")
    whole[:, :n], whole[:, n:2 * n] = torch.as_tensor(x), torch.as_tensor(r)
    at, dw, s = whole.data_ptr(), torch.as_tensor(w).cuda(), torch.empty(rows, device="cuda")
    h = whole[:, :n] + whole[:, n:2 * n]
    L.add_rms_norm_q8(at, at + 4 * n, at + 8 * n, dw.data_ptr(), 1e-6, rows, n, at + 12 * n, s.data_ptr(), x_stride=step,
                      residual_stride=step, h_stride=step, q_stride=4 * step, stream=stream())
    torch.cuda.synchronize()
    q = whole.view(torch.int8)[:, 12 * n:13 * n]
    assert torch.equal(whole[:, 2 * n:3 * n], h)
    check_rows(q, s, *ref.norm_q8(f64(h), w, 1e-6))
    L.swiglu_q8(at, at + 4 * n, rows, n, at + 8 * n, s.data_ptr(), gate_stride=step, up_stride=step, q_stride=4 * step, stream=stream())
    torch.cuda.synchronize()
    check_rows(whole.view(torch.int8)[:, 8 * n:9 * n], s, *ref.swiglu_q8(f64(whole[:, :n]), f64(whole[:, n:2 * n])))
    assert bool((whole[:, -3:] == 77.0).all())
