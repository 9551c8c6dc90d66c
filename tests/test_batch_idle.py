"""Streams over the paged 4-bit cache that were released and have no prompt yet: the
others go on without them, on the pages they gave back."""
import ctypes

import numpy as np
import pytest

from emberllm_b200 import EmberBatch, Sampler

from .test_batch_kv4 import ember, prompts, run      # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu
ints = lambda v: (ctypes.c_int * len(v))(*v)


def test_the_others_go_on_in_a_pool_that_is_just_large_enough(ember):
    ps = prompts(ember, [70, 60, 150], 4)
    alone = [run(ember, [p], 45, kv4=True) for p in ps]
    # 2 + 1 + 3 pages; 45 steps take the third stream to 195 positions, its fourth page
    b = EmberBatch(ember, 3, ctx=200, max_steps=45, kv4=True, pages=6)
    lib, dev = b.lib, b.lib.ember_batch_cuda(b.b)
    firsts = [b.prefill(i, p) for i, p in enumerate(ps)]
    assert [lib.ember_cuda_batch_idle(dev, i) for i in range(-1, 4)] == [0] * 5
    b.release(1)
    assert [lib.ember_cuda_batch_idle(dev, i) for i in range(3)] == [0, 1, 0]
    toks, lg = b.greedy([firsts[0], -12345, firsts[2]], [70, 2 ** 31 - 1, 150], 45, logits=True)
    lg = np.ctypeslib.as_array(lg).reshape(3, ember.vocab)
    for i in (0, 2):
        assert [t[i] for t in toks] == [t[0] for t in alone[i][1]]
        assert np.array_equal(lg[i], alone[i][2][0])
    assert all(t[1] == -1 for t in toks) and (lg[1] == 0).all()
    # no page is left for its prompt; with the third stream's there are
    assert lib.ember_cuda_batch_prefill(dev, 1, ints(ps[1]), 60, None) == 1
    assert b"pages" in lib.ember_cuda_error() and lib.ember_cuda_batch_idle(dev, 1) == 1
    b.release(2)
    assert b.prefill(1, ps[1]) == alone[1][0][0] and lib.ember_cuda_batch_idle(dev, 1) == 0
    b.release(0)
    toks = b.greedy([0, firsts[1], 0], [0, 60, 0], 45)
    assert [t[1] for t in toks] == [t[0] for t in alone[1][1]]
    assert all(t[0] == t[2] == -1 for t in toks)
    b.close()


def test_drawn_steps_and_refusals(ember):
    ps = prompts(ember, [20, 30, 65], 6)
    u = np.random.default_rng(2).random((6, 3), dtype=np.float32)
    sm = [Sampler(0.8), Sampler(1.0), Sampler(0.9, 0.9)]
    b = EmberBatch(ember, 3, ctx=96, max_steps=200, kv4=True)
    dev = b.lib.ember_batch_cuda(b.b)
    firsts = [b.prefill(i, p) for i, p in enumerate(ps)]
    want = b.sample(firsts, [20, 30, 65], 6, sm, u)
    for i, p in enumerate(ps):
        b.prefill(i, p)
    b.release(1)
    sm[1].set_penalties(repeat_penalty=1.3)                     # not looked at
    u[:, 1] = np.nan
    got = b.sample([firsts[0], -1, firsts[2]], [20, -1, 65], 6, sm, u)
    assert [[t[0], t[2]] for t in got] == [[t[0], t[2]] for t in want] and all(t[1] == -1 for t in got)
    # a live stream's numbers are checked as ever; nobody at all is a step, too
    assert b.lib.ember_cuda_batch_greedy(dev, ints([1, 1, 1]), ints([20, 0, -1]), 1, None, None) == 1
    b.release(0)
    b.release(2)
    b.release(2)
    assert b.greedy([0] * 3, [0] * 3, 3) == [[-1] * 3] * 3
    assert b.lib.ember_cuda_batch_greedy(dev, ints([0] * 3), ints([0] * 3), 97, None, None) == 1
    for i, p in enumerate(ps):
        assert b.prefill(i, p) == firsts[i]
    b.close()


def test_contexts_that_no_table_can_hold_are_refused(ember):
    """at the C entry: a status, never an exception or an overflow"""
    b = EmberBatch(ember, 1, ctx=64, max_steps=1, kv4=True)
    lib = b.lib
    model = ctypes.cast(ctypes.c_void_p(lib.ember_batch_cuda(b.b)), ctypes.POINTER(ctypes.c_void_p))[0]   # its first member
    new, out = lib.ember_cuda_batch_new_kv4, ctypes.c_void_p(1)
    new.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 5 + [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    rope = (ctypes.c_float * (64 * 64 * 2))()
    for streams, ctx, pages in ((1, 0, 10), (2, -5, 10), (1, 2 ** 31 - 1, 10), (512, 2 ** 31 - 100, 10), (3, 2 ** 30, 0),
                                (0, 64, 0), (513, 64, 0), (1, 64, -1), (1, 64, 2 ** 26)):
        assert new(model, streams, ctx, pages, 0, 0, rope, 1, ctypes.byref(out)) == 1
        assert out.value is None and b"batch" in lib.ember_cuda_error()
    assert new(model, 2, 64, 0, 0, 0, rope, 1, ctypes.byref(out)) == 0 and out.value
    lib.ember_cuda_batch_free.argtypes = [ctypes.c_void_p]
    lib.ember_cuda_batch_free(out)
    b.close()
