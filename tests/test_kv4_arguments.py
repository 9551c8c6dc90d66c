"""What the Python face of the 4-bit cache and of the draws refuses before the library
sees it: ValueError, as its documentation says. (On the CPU: whatever passes the
checks ends at the library's own, for host memory.)"""
import pytest

from emberllm_b200 import Kv4Cache, sample_rows

from . import helpers as H
from .test_kv4 import cpu_call

torch = pytest.importorskip("torch")
I32 = torch.int32


@pytest.mark.parametrize("workspace", [
    torch.empty(1, dtype=torch.uint8).expand(1 << 20),             # a byte that looks like a million
    torch.empty(1 << 20, dtype=torch.uint8)[::2], torch.empty(64, 64)[:, :32]])
def test_a_workspace_with_holes(workspace):
    with pytest.raises(ValueError, match="workspace"):
        cpu_call(workspace=workspace)
    with pytest.raises(RuntimeError, match="device memory"):
        cpu_call(workspace=workspace.contiguous())


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(192)), dict(q=torch.zeros(3, 256)), dict(q=torch.zeros(1, 3, 4, 64)), dict(lens=torch.zeros(3, 1, dtype=I32)),
    dict(lens=torch.tensor(3, dtype=I32)),
    dict(max_q=1 << 40), dict(max_kv=1 << 31), dict(window=1 << 31), dict(sinks=-1 << 40), dict(max_q=1.5)])
def test_shapes_and_numbers_that_do_not_fit(change):
    with pytest.raises(ValueError):
        cpu_call(**change)


def test_a_scale_that_is_infinite_in_single_precision():
    with pytest.raises((ValueError, RuntimeError)):
        cpu_call(scale=1e39)


@pytest.mark.parametrize("args", [((1 << 32) + 4, 16, 2, 64), (4, (1 << 32) + 16, 2, 64), (4, 16, 2, 64 - (1 << 32))])
def test_sizes_are_not_taken_modulo_a_word(args):
    H.ensure_built()
    with pytest.raises(ValueError):
        Kv4Cache.nbytes(*args)


def test_of_stores_caches_and_draws():
    H.ensure_built()
    buf = torch.zeros(Kv4Cache.nbytes(4, 16, 2, 64), dtype=torch.uint8)
    cache = Kv4Cache(buf, 4, 16, 2, 64)
    k = torch.zeros(1, 2, 64)
    for lens, table, kw in ((torch.zeros(1, 1, dtype=I32), torch.zeros(1, 1, dtype=I32), {}),
                            (torch.zeros(1, dtype=I32), torch.zeros(1, dtype=I32), {}),
                            (torch.zeros(1, dtype=I32), torch.zeros(1, 1, dtype=I32), dict(max_q=1 << 33))):
        for fn in (cache.store, cache.read):
            with pytest.raises(ValueError):
                fn(k, k, None, lens, table, **kw)
    with pytest.raises(ValueError):
        Kv4Cache(buf[:1].expand(buf.numel()), 4, 16, 2, 64)
    for logits in (torch.zeros(8), torch.zeros(2, 2, 8), torch.zeros(2, 8).t()):
        with pytest.raises(ValueError):
            sample_rows(logits, torch.zeros(2, dtype=I32), torch.zeros(2))
