"""A device wait of the many-row attention that runs out: the call ends, its rows are
NaN, the status says so once and the context stays usable. The tests make the wait for
the keys one for an arrival that never comes, with a limit of 200 microseconds."""
import ctypes

import numpy as np
import pytest

from emberllm_b200 import Ember, EmberBatch, Kv4Cache, synth

from . import helpers as H
from .test_kv4_many_rows import ALL, MANY_1, kernel, make

torch = pytest.importorskip("torch")


def test_status_is_refused_on_host_memory():
    H.ensure_built()
    cache = Kv4Cache(torch.zeros(Kv4Cache.nbytes(4, 16, 2, 64), dtype=torch.uint8), 4, 16, 2, 64)
    with pytest.raises(RuntimeError, match="device memory"):
        cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
def test_a_wait_that_runs_out_is_reported(monkeypatch, shape, dtype):
    p, q = make(shape, dtype)
    first = p.attend(q)
    p.cache.check()
    monkeypatch.setenv("EMBER_KV4_LOST_KEYS_US", "200")
    got = p.attend(q)
    monkeypatch.delenv("EMBER_KV4_LOST_KEYS_US")
    with pytest.raises(RuntimeError, match="wait timed out"):
        p.cache.check()
    p.cache.check()                                   # said once
    assert torch.isnan(got).all()
    for _ in range(3):
        assert torch.equal(p.attend(q), first)
    p.cache.check(torch.cuda.Stream().cuda_stream)


@pytest.mark.gpu
def test_a_prompt_whose_wait_runs_out_fails(monkeypatch):
    assert kernel(torch.float32, 512, 16, 8, 64, 1) == MANY_1
    monkeypatch.setitem(synth.CONFIGS, "tiny-heads", dict(
        dim=256, hidden_dim=512, n_layers=2, n_heads=16, n_kv_heads=8, head_dim=64, vocab_size=512, max_seq_len=2048,
        rope_theta=1e6, norm_eps=1e-6, rope_style=synth.ROPE_NEOX, tied=True, qk_norm=True, bias=False, quant="q8_0"))
    H.ensure_built()
    e = Ember(synth.ensure_model("tiny-heads"))
    b = EmberBatch(e, 2, max_steps=1, kv4=True)
    ids = [int(t) for t in np.random.default_rng(1).integers(0, 512, 600)]
    want = b.prefill(0, ids)
    dev, arr = b.lib.ember_batch_cuda(b.b), (ctypes.c_int * 600)(*ids)
    monkeypatch.setenv("EMBER_KV4_LOST_KEYS_US", "200")
    assert b.lib.ember_cuda_batch_prefill(dev, 1, arr, 600, None) == 1
    assert b"wait timed out" in b.lib.ember_cuda_error()
    monkeypatch.delenv("EMBER_KV4_LOST_KEYS_US")
    assert b.prefill(1, ids) == want
    b.close()
    e.close()
