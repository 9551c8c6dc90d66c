"""Calls without a stream go where torch's own operations go: inside
``torch.cuda.stream(s)`` they wait for what s still has to do, and a graph captures them."""
import pytest

from emberllm_b200 import kv4, sample_rows

from .test_kv4 import Paged, plain_values

torch = pytest.importorskip("torch")


def test_arrays_that_torch_has_on_the_host_or_does_not_know():
    assert kv4._on(None, torch.zeros(1)) == 0 and kv4._on(None, object()) == 0 and kv4._on(7, torch.zeros(1)) == 7


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 330])
def test_calls_wait_for_the_current_stream(ql):
    p = Paged([400], [ql], 64, 8, 128, seed=1)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(400, 8, 128, generator=g).cuda() for _ in range(2))
    q = torch.randn(ql, 16, 128, generator=g).cuda()
    x = torch.randn(4, 5000, generator=g).cuda()
    u = torch.rand(4, generator=g).cuda()
    late = [torch.zeros_like(t) for t in (k, v, q, x, u)]
    kb, vb, out, tok = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(q), torch.zeros(4, dtype=torch.int32, device="cuda")
    ws = p.workspace(16)
    args = (p.full, p.kv_len, p.table, 400)

    def calls():
        for t, src in zip(late, (k, v, q, x, u)):
            t.copy_(src)
        p.cache.store(late[0], late[1], *args)
        p.cache.read(kb, vb, *args)
        p.cache.attention(late[2], out, p.start, p.kv_len, p.table, ql, 400, workspace=ws)
        sample_rows(late[3], tok, late[4])
    torch.cuda.synchronize()
    calls()
    torch.cuda.synchronize()
    want = [t.clone() for t in (kb, vb, out, tok)]
    assert torch.equal(kb.double(), plain_values(k))
    s = torch.cuda.Stream()
    for t in late + [kb, vb, out, tok]:
        t.zero_()
    p.buf.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(40_000_000)              # some 20 ms of work before the inputs are there
        calls()
        p.cache.check()                            # (waits for s)
        assert s.query()
    assert all(torch.equal(a, b) for a, b in zip((kb, vb, out, tok), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for t in late + [kb, vb, out, tok]:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((kb, vb, out, tok), want))
