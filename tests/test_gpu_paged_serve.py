"""The serving operators together (dpuf_b200.paged_serve) against the engine on the same model."""
import numpy as np
import pytest
import torch

from dpuf_b200 import engine, model as mdl

pytestmark = pytest.mark.gpu


def close(a, b):
    """As for the fp16 engine cache: every layer re-quantizes its activations to int8 blocks, which turns
    rounding differences into whole steps on a few elements; the difference's RMS stays within 5 %."""
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    rms = np.sqrt(np.mean(a * a))
    rd = np.sqrt(np.mean((a - b) ** 2))
    assert rd <= 0.05 * rms, rd / rms


@pytest.mark.parametrize("kv", ["float32", "float16"])
@pytest.mark.parametrize("shape", ["TINY", "TINY_G3", "TINY_MHA"])
def test_steps_match_the_engine(shape, kv):
    from dpuf_b200 import paged_serve

    m = mdl.SyntheticModel(getattr(mdl, shape), seed=4, norm_jitter=0.1)
    ref = engine.CudaTransformerEngine(m)
    paged = paged_serve.PagedModel(m, 40, kv_dtype=getattr(torch, kv))
    try:
        prompts = [mdl.prompt_ids(n, m.shape.vocab, 30 + n) for n in (1, 37, 90)]
        seqs = [paged.open() for _ in prompts]
        # the first step holds whole prompts and, of the longest, a chunk; the second the rest beside a token
        logits = paged.step([(s, list(p[:60])) for s, p in zip(seqs, prompts)]).cpu().numpy()
        want = []
        for i, p in enumerate(prompts):
            ref.set_slot(i)
            ref.reset_slot(i)
            want.append(ref.forward_batch(p[:60], 0)[0])
            close(want[i], logits[i])
        feed = [[int(np.argmax(w))] for w in want]
        feed[2] = list(prompts[2][60:])
        logits = paged.step(list(zip(seqs, feed))).cpu().numpy()
        for i, p in enumerate(prompts):
            ref.set_slot(i)
            close(ref.forward_batch(feed[i], min(len(p), 60))[0], logits[i])
        used = 40 - len(paged.free)
        paged.close(seqs[1])
        assert 40 - len(paged.free) < used
    finally:
        paged.release()
        ref.close()


def test_generate_frees_its_pages_and_repeats():
    from dpuf_b200 import paged_serve

    m = mdl.SyntheticModel(mdl.TINY, seed=2)
    paged = paged_serve.PagedModel(m, 60)
    try:
        prompts = [mdl.prompt_ids(n, m.shape.vocab, n) for n in (3, 130, 20)]
        a = paged_serve.generate(paged, prompts, 8, 0.9, 40, 0.95, 0.01, seed=5)
        assert len(paged.free) == 60 and [len(x) for x in a] == [8] * 3
        # other pages (the free list's order has changed), the same tokens
        assert a == paged_serve.generate(paged, prompts, 8, 0.9, 40, 0.95, 0.01, seed=5)
        greedy = paged_serve.generate(paged, prompts, 4)
        assert all(0 <= t < m.shape.vocab for x in greedy for t in x)
        with pytest.raises(RuntimeError):
            paged.step([(paged.open(), [1] * 500), (paged.open(), [1] * 500)])
        with pytest.raises(ValueError):
            paged.step([(0, [])])
    finally:
        paged.release()


def test_generate_frees_its_pages_where_a_step_fails():
    from dpuf_b200 import paged_serve

    m = mdl.SyntheticModel(mdl.TINY, seed=2)
    paged = paged_serve.PagedModel(m, 12)
    try:
        prompts = [mdl.prompt_ids(n, m.shape.vocab, n) for n in (3, 60, 20)]
        for error, bad in ((ValueError, prompts + [[]]), (RuntimeError, prompts + [prompts[1]] * 3)):
            with pytest.raises(error):
                paged_serve.generate(paged, bad, 4)
            assert len(paged.free) == 12 and not paged.pages and not paged.length
        with pytest.raises(ValueError):
            paged_serve.generate(paged, prompts, 4, chunk=0)
        assert len(paged.free) == 12
        assert [len(x) for x in paged_serve.generate(paged, prompts, 4)] == [4] * 3
    finally:
        paged.release()


def test_a_step_says_that_a_wait_gave_up():
    """The attention's error word set, as a kernel that gave up leaves it: the step raises, and can be repeated."""
    from dpuf_b200 import paged_serve

    m = mdl.SyntheticModel(mdl.TINY, seed=2)
    paged = paged_serve.PagedModel(m, 12)
    try:
        s = paged.open()
        want = paged.step([(s, [5, 6, 7])])
        paged.close(s)
        s = paged.open()
        paged.workspace[:1] = 1
        with pytest.raises(RuntimeError, match="gave up"):
            paged.step([(s, [5, 6, 7])])
        assert paged.length[s] == 0
        assert torch.equal(want, paged.step([(s, [5, 6, 7])]))
    finally:
        paged.release()


def test_command_line(capsys):
    from dpuf_b200 import paged_serve

    paged_serve.main(["--sequences", "2", "--tokens", "3"])
    assert capsys.readouterr().out.count("sequence ") == 2
