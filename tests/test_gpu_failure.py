"""Failure detection on the device without a GPU fault.

Every wait inside the persistent step (a tagged word another CTA writes, a
bulk copy's barrier) is bounded: when it runs out, the kernel sets the
context's status word, gives up its remaining waits at once and runs to its
end, and the step returns -1.  Here a wait is made to run out on purpose --
ecu_inject_wait_timeout makes the next step wait for an input word that no
phase writes (a flag that nothing sets) -- with the limit shortened to
0.2 s.  The test checks the -1, the message, the time it took, and that the
same context then produces the oracle's greedy tokens again.  (The
reference's failure paths are host retries and aborts, src/shard.c:533-545.)
"""
import time

import numpy as np
import pytest

from distcomp_b200 import synth

pytestmark = pytest.mark.gpu


def test_wait_runs_out_and_context_recovers(eng, oracle_port, model_buf):
    import oracle
    key = "mini-q4"
    s = synth.spec(key)
    buf = model_buf(key)
    prompt = synth.prompt_tokens(6, s.n_vocab, seed=3)
    want = oracle.greedy(oracle_port, buf, prompt, 8)
    c = eng.LlmCtx(eng.GgufModel(buf), eng.STAGE_FULL, n_ctx=64)
    assert c.path() == "persistent"
    assert c.generate(prompt, 8) == want
    eng.set_wait_ns(200_000_000)
    try:
        out = np.zeros(s.n_embd + 1, dtype=np.float32)
        for _ in range(2):                          # twice: the recovery is complete
            c.reset()
            c.inject_wait_timeout()
            t0 = time.perf_counter()
            assert c.forward(prompt[0], out) == -1
            dt = time.perf_counter() - t0
            assert "bounded wait" in eng.last_error()
            assert 0.15 <= dt < 10.0, dt
            c.reset()
            assert c.generate(prompt, 8) == want
    finally:
        eng.set_wait_ns(2_000_000_000)
    c.close()


def test_a_warp_that_comes_late_to_every_phase(eng, model_buf):
    """A warp that reaches each phase long after the next phase's descriptor has landed: the step takes longer, and its
    token, state and logits are the same bits."""
    c = eng.LlmCtx(eng.GgufModel(model_buf("mini-q4", n_layer=4)), eng.STAGE_FULL, n_ctx=64)
    assert c.path() == "persistent"
    eng.set_wait_ns(200_000_000)                     # a step that stood still would give up after this
    try:
        outs = []
        for late in (False, True, True, False):
            c.reset()
            steps = []
            for t in (3, 9, 27, 81):
                out = np.zeros(c.n_embd + 1, dtype=np.float32)
                if late:
                    c.inject_late_warp()
                assert c.forward(t, out) == 0, eng.last_error()
                steps.append((out.copy(), c.logits().copy()))
            outs.append(steps)
        for steps in outs[1:]:
            for (a, la), (b, lb) in zip(outs[0], steps):
                assert np.array_equal(a.view(np.uint32), b.view(np.uint32)) and np.array_equal(la.view(np.uint32), lb.view(np.uint32))
    finally:
        eng.set_wait_ns(2_000_000_000)
    c.close()
    c = eng.LlmCtx(eng.GgufModel(model_buf("mini-q8")), eng.STAGE_FULL, n_ctx=16)
    with pytest.raises(eng.EngineError, match="4 query heads of 128"):
        c.inject_late_warp()
    c.close()


def test_injection_needs_the_persistent_step(eng, model_buf, monkeypatch):
    monkeypatch.setenv("ECU_MEGA", "0")
    c = eng.LlmCtx(eng.GgufModel(model_buf("mini-q4")), eng.STAGE_FULL, n_ctx=16)
    with pytest.raises(eng.EngineError, match="persistent"):
        c.inject_wait_timeout()
    with pytest.raises(eng.EngineError, match="positive"):
        eng.set_wait_ns(0)
    c.close()


@pytest.fixture
def short_wait(eng):
    eng.set_wait_ns(100_000_000)
    yield
    eng.set_wait_ns(2_000_000_000)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [40, 700])             # all keys requested at once; keys waiting for a place of the ring
def test_prompt_attention_gives_up_and_reports(eng, short_wait, hd, n):
    """Keys that are never copied: the rows become NaN, the status reports it once, and the next call is right."""
    import torch

    from distcomp_b200 import kv4
    g = torch.Generator().manual_seed(n + hd)
    q, k, v = (torch.randn(n, h, hd, generator=g).half().cuda() for h in (8, 2, 2))
    want = kv4.prompt_attention(q, k, v, [0, n])
    kv4.prompt_status()
    for _ in range(2):
        eng.inject_prompt_timeout()
        t0 = time.perf_counter()
        out = kv4.prompt_attention(q, k, v, [0, n])
        with pytest.raises(eng.EngineError, match="bounded wait"):
            kv4.prompt_status()
        dt = time.perf_counter() - t0
        assert 0.08 <= dt < 5.0, dt
        assert torch.isnan(out).all()
        assert torch.equal(kv4.prompt_attention(q, k, v, [0, n]), want)
        kv4.prompt_status()


def test_batch_reports_a_prompt_that_gave_up(eng, short_wait, model_buf):
    """The feed fails, the sequences keep what they held, and the batch goes on as one that never failed."""
    m = eng.GgufModel(model_buf("mini-q4"))
    base = eng.LlmCtx(m, eng.STAGE_FULL)
    a, b = eng.LlmBatch(base, 3, 9), eng.LlmBatch(base, 3, 9)
    for x in (a, b):
        x.feed([0, 1], [[5] * 40, [7, 8, 9]])
    eng.inject_prompt_timeout()
    with pytest.raises(eng.EngineError, match="bounded wait"):
        a.feed([0, 1, 2], [[3], [4] * 70, [6] * 30])
    assert [a.length(s) for s in range(3)] == [40, 3, 0] and a.used() == b.used()
    for _ in range(2):
        (pa, la), (pb, lb) = (x.feed([0, 1, 2], [[3], [4] * 20, [6] * 30], logits=True) for x in (a, b))
        assert pa == pb and np.array_equal(la, lb)


def test_prefill_reports_a_prompt_that_gave_up(eng, short_wait, model_buf, monkeypatch):
    monkeypatch.setenv("ECU_PF_ATTN", "2")
    c = eng.LlmCtx(eng.GgufModel(model_buf("mini-q4")), eng.STAGE_FULL, n_ctx=128)
    prompt = [3, 9, 27] * 20
    want = c.prefill(prompt)
    c.reset()
    eng.inject_prompt_timeout()
    with pytest.raises(eng.EngineError, match="bounded wait"):
        c.prefill(prompt)
    c.reset()
    assert c.prefill(prompt) == want
    c.close()


def test_batch_whose_pool_update_fails(eng, model_buf):
    """A feed that the pool refuses on the device changes nothing and can be made again."""
    m = eng.GgufModel(model_buf("mini-q4"))
    b = eng.LlmBatch(eng.LlmCtx(m, eng.STAGE_FULL), 3, 9)
    b.feed([0, 1], [[5] * 64, [7, 8, 9]])
    b.fork([1], [2])
    want = [b.length(s) for s in range(3)], b.used()
    assert eng.lib().ecu_kv_inject_failure(b.kv, 0) == 0
    with pytest.raises(eng.EngineError, match="injected"):
        b.feed([0, 2, 1], [[3], [4], [6] * 70])
    assert ([b.length(s) for s in range(3)], b.used()) == want
    first = b.feed([0, 2, 1], [[3], [4], [6] * 70])
    b.free([0, 1, 2])
    b.feed([0, 1, 2], [[5] * 64, [7, 8, 9], [7, 8, 9]])
    assert b.feed([0, 2, 1], [[3], [4], [6] * 70]) == first
