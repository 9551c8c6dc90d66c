"""Streams over a paged 4-bit cache and drawn steps (ember_batch_new_kv4,
ember_batch_sample): store, attention and sampling run together as a batch uses them."""
import ctypes

import numpy as np
import pytest

from emberllm_b200 import Ember, EmberBatch, Sampler, _lib, synth

from . import helpers as H
from .test_sample_rows import plain

pytestmark = pytest.mark.gpu
FP = ctypes.POINTER(ctypes.c_float)


@pytest.fixture(scope="module", params=["tiny-qwen3", "tiny-llama", "tiny-mqa"])
def ember(request):
    H.ensure_built()
    e = Ember(synth.ensure_model(request.param))
    yield e
    e.close()


def prompts(ember, lens, seed=0):
    rng = np.random.default_rng(seed)
    return [[int(t) for t in rng.integers(0, ember.vocab, n)] for n in lens]


def start(b, ps):
    return [b.prefill(i, p) for i, p in enumerate(ps)], [len(p) for p in ps]


def run(ember, ps, steps, **kw):
    b = EmberBatch(ember, len(ps), ctx=200, max_steps=steps, **kw)
    firsts, pos = start(b, ps)
    toks, lg = b.greedy(firsts, pos, steps, logits=True)
    b.close()
    return firsts, toks, np.ctypeslib.as_array(lg).reshape(len(ps), ember.vocab).copy()


def drawn_step(b, toks, pos, samplers, u, vocab):
    """one drawn step with its logits"""
    n = len(toks)
    s = (_lib.EmberSampleParams * n)(*[x.params() for x in samplers])
    out, lg = (ctypes.c_int * n)(), (ctypes.c_float * (n * vocab))()
    rc = b.lib.ember_cuda_batch_sample(b.lib.ember_batch_cuda(b.b), (ctypes.c_int * n)(*toks), (ctypes.c_int * n)(*pos), 1, s,
                                       (ctypes.c_float * n)(*u), out, ctypes.cast(lg, FP))
    assert rc == 0, b.lib.ember_cuda_error()
    return list(out), np.ctypeslib.as_array(lg).reshape(n, vocab).copy()


LENS = [1, 5, 63, 64, 65, 17, 130, 2, 30, 100]


def test_streams_do_not_depend_on_each_other(ember):
    """a stream's tokens and last logits, bit for bit, alone and among others"""
    ps = prompts(ember, LENS)
    firsts, toks, lg = run(ember, ps, 20, kv4=True)
    for i in (0, 3, 6, 9):
        f, t, l = run(ember, [ps[i]], 20, kv4=True)
        assert f == [firsts[i]] and [x[0] for x in t] == [x[i] for x in toks]
        assert np.array_equal(l[0].view(np.uint32), lg[i].view(np.uint32))


def test_near_the_exact_cache(ember):
    """a 4-bit value is off by half a step, 8% of a value in the mean; the residual
    stream carries the rest, so the logits keep their direction"""
    ps = prompts(ember, LENS, 3)
    exact = EmberBatch(ember, len(ps), ctx=200, max_steps=1)
    quant = EmberBatch(ember, len(ps), ctx=200, max_steps=1, kv4=True)
    rows = []
    for b in (exact, quant):
        start(b, ps)
        _, lg = b.greedy([7] * len(ps), [len(p) for p in ps], 1, logits=True)
        rows.append(np.ctypeslib.as_array(lg).reshape(len(ps), ember.vocab).astype(np.float64))
        b.close()
    a, q = rows
    cos = (a * q).sum(1) / np.linalg.norm(a, axis=1) / np.linalg.norm(q, axis=1)
    assert cos.min() > 0.95


def test_windows(ember):
    ps = prompts(ember, LENS, 1)
    want = run(ember, ps, 8, kv4=True)
    wide = run(ember, ps, 8, kv4=True, window=200, sinks=3)
    assert want[0] == wide[0] and want[1] == wide[1] and np.array_equal(want[2], wide[2])
    narrow = run(ember, ps, 8, kv4=True, window=4, sinks=1)
    assert np.isfinite(narrow[2]).all() and not np.array_equal(narrow[2][6], want[2][6])


def test_pages_are_taken_given_back_and_run_out(ember):
    ps = prompts(ember, [100, 60, 130], 2)
    want = run(ember, ps, 10, kv4=True)
    # 100 + 10 positions: 2 pages; 70: 2; 140: 3
    b = EmberBatch(ember, 3, ctx=200, max_steps=10, kv4=True, pages=7)
    for _ in range(3):
        firsts, pos = start(b, ps)
        toks, _ = b.greedy(firsts, pos, 10, logits=True)
        assert firsts == want[0] and toks == want[1]
        for i in (1, 2, 0):
            b.release(i)
    b.close()
    b = EmberBatch(ember, 3, ctx=200, max_steps=10, kv4=True, pages=6)
    firsts, pos = start(b, ps)
    ints = lambda v: (ctypes.c_int * len(v))(*v)
    dev = b.lib.ember_batch_cuda(b.b)
    assert b.lib.ember_cuda_batch_greedy(dev, ints(firsts), ints(pos), 10, None, None) == 1
    assert b"pages" in b.lib.ember_cuda_error()
    assert b.lib.ember_cuda_batch_greedy(dev, ints(firsts), ints(pos), 2, None, None) == 0   # 2 + 1 + 3 pages
    b.close()


@pytest.mark.parametrize("kv4", [False, True])
def test_drawn_steps(ember, kv4):
    ps = prompts(ember, LENS, 5)
    n = len(ps)
    b = EmberBatch(ember, n, ctx=200, max_steps=8, kv4=kv4)
    # temperature 0: the greedy run
    firsts, pos = start(b, ps)
    greedy = b.greedy(firsts, pos, 8)
    firsts, pos = start(b, ps)
    u = np.random.default_rng(1).random((8, n), dtype=np.float32)
    assert b.sample(firsts, pos, 8, [Sampler() for _ in range(n)], u) == greedy
    # settings of every kind: each step draws from its logits; eight at once are the same
    sm = [Sampler(0.5 + 0.1 * i, (1.0, 0.9, 0.5)[i % 3], (0, 20, 0, 3)[i % 4]) for i in range(n)]
    for i in (2, 5):
        sm[i].set_penalties(min_p=0.05)
    firsts, pos = start(b, ps)
    toks, steps = firsts, []
    for t in range(8):
        toks, lg = drawn_step(b, toks, [p + t for p in pos], sm, u[t], ember.vocab)
        want = [plain(lg[i], u[t, i], sm[i].temperature, sm[i].top_k, sm[i].top_p, sm[i].min_p) for i in range(n)]
        assert toks == want
        steps.append(toks)
    firsts, pos = start(b, ps)
    assert b.sample(firsts, pos, 8, sm, u) == steps
    b.close()


def test_refusals(ember):
    b = EmberBatch(ember, 2, ctx=64, max_steps=4, kv4=True)
    dev, lib = b.lib.ember_batch_cuda(b.b), b.lib
    ints = lambda *v: (ctypes.c_int * len(v))(*v)
    u = (ctypes.c_float * 8)()

    def sample(toks=(1, 2), pos=(3, 3), n=1, **kw):
        sp = [Sampler(1.0), Sampler(1.0)]
        for k, v in kw.items():
            setattr(sp[1], k, v)
        s = (_lib.EmberSampleParams * 2)(*[x.params() for x in sp])
        return lib.ember_cuda_batch_sample(dev, ints(*toks), ints(*pos), n, s, u, None, None)
    assert sample() == 0
    assert sample(toks=(1, ember.vocab)) and sample(toks=(-1, 0)) and sample(pos=(0, 64)) and sample(pos=(0, 2 ** 31 - 1))
    assert sample(n=0) and sample(n=5) and sample(repeat_penalty=1.1) and sample(temperature=float("nan"))
    b.close()
    e = EmberBatch(ember, 2, ctx=64, max_steps=4)
    dev = lib.ember_batch_cuda(e.b)
    assert sample() == 1 and b"streams" in lib.ember_cuda_error()
    assert lib.ember_cuda_batch_release(dev, 0) == 1
    e.close()
