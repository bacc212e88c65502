"""A kernel's shared-memory limit belongs to the process: contexts of several
sizes, used one after another and from several threads, keep working."""
import threading

import numpy as np
import pytest

import lal_b200 as L
import oracle
from lal_b200 import synth

pytestmark = pytest.mark.gpu


def gpt2_step(vocab, n_embd):
    """One step of the GPT-2 tail, whose kernels' shared memory grows with the
    vocabulary and the width, against the oracle's."""
    cfg = synth.CONFIGS["c1_gpt2"].with_(vocab=vocab, n_embd=n_embd, hist=8)
    q, s = oracle.quantize_rows(synth.lm_head_f32(cfg), "port")
    t = L.DecodeTail(vocab, n_embd, max_top_k=40, history_cap=8, sampler=L.LAL_SAMPLER_GPT2)
    t.load_lm_head_q8(q, s)
    t.set_sampling([0.9], [40], [1.0])
    t.set_history(0, np.zeros(0, np.int32))
    port = oracle.Gpt2PortLoop(q, s, [], 8, 0.9, 40, 1.0)
    x = synth.hidden(cfg, 0)
    assert int(t.step(x, np.array([0.25], np.float32))[0]) == port.step(x[0], np.float32(0.25))[0]
    t.close()


def test_gpt2_contexts_of_growing_size():
    for vocab, n_embd in ((700, 64), (5003, 768), (20011, 1600), (700, 64), (20011, 1600)):
        gpt2_step(vocab, n_embd)


def test_gpt2_contexts_of_two_threads():
    """A thread's first, small launch does not lower what another's needs."""
    gpt2_step(20011, 1600)
    failed = []

    def other():
        try:
            gpt2_step(700, 64)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    for _ in range(2):
        th = threading.Thread(target=other)
        th.start()
        th.join()
        gpt2_step(20011, 1600)
    assert not failed, failed
