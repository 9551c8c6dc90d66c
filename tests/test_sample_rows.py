"""One draw per row (ember_cuda_sample_rows) against a plain 64-bit implementation
of its definition. Tokens are whole numbers and have to be equal."""
import numpy as np
import pytest

from emberllm_b200 import sample_rows

from . import helpers as H

torch = pytest.importorskip("torch")


def plain(logits, u, temperature, top_k, top_p, min_p):
    """one row, numpy float64; sorted by (logit descending, index ascending)"""
    x = logits.astype(np.float32).copy()
    x[np.isnan(x)] = -np.inf
    order = np.argsort(-x, kind="stable")
    mx = x[order[0]]
    if mx == -np.inf:
        return 0
    if not temperature > 0:
        return int(order[0])
    l = x[order].astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l == mx, 1.0, np.where(l == -np.inf, 0.0, np.exp((l - np.float64(mx)) / np.float64(np.float32(temperature)))))
    run = np.cumsum(w)
    keep = len(x)
    if 0 < top_k < keep:
        keep = top_k
    if 0 < min_p < 1:
        keep = min(keep, int((w >= np.float64(np.float32(min_p))).sum()))
    if 0 < top_p < 1:
        keep = min(keep, int((run < np.float64(np.float32(top_p)) * run[-1]).sum()) + 1)
    u = np.float32(u)
    r = (0.0 if not u > 0 else min(float(u), 1.0)) * run[keep - 1]
    i = int((run <= r).sum())
    last = int(np.nonzero(w[:keep])[0][-1])
    return int(order[min(i, last)])


def draw(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    n = x.shape[0]
    dev = lambda v, t: None if v is None else torch.tensor(np.broadcast_to(v, (n,)).copy(), dtype=t).cuda()
    out = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    sample_rows(x, out, dev(u, torch.float32), dev(temperature, torch.float32), dev(top_k, torch.int32),
                dev(top_p, torch.float32), dev(min_p, torch.float32))
    got = out.cpu().numpy()
    xs = x.float().cpu().numpy()
    b = lambda v, d: np.broadcast_to(d if v is None else v, (n,))
    want = [plain(xs[i], b(u, 0)[i], b(temperature, 1.0)[i], int(b(top_k, 0)[i]), b(top_p, 1.0)[i], b(min_p, 0.0)[i])
            for i in range(n)]
    assert got.tolist() == want
    return got


def logits(n, vocab, seed=0, dtype=torch.float32, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, vocab, generator=g) * scale).to(dtype).cuda()


def us(n, seed=1):
    return np.random.default_rng(seed).random(n, dtype=np.float32)


# ---------------------------------------------------------------------- CPU ----

@pytest.mark.parametrize("change,exc", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), ValueError),
    (dict(logits=torch.zeros(2, 16)[:, ::2]), ValueError),
    (dict(logits=torch.zeros(8)), ValueError),
    (dict(out=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(out=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(u=torch.zeros(2, dtype=torch.float64)), ValueError),
    (dict(top_k=torch.zeros(2)), ValueError),
    (dict(temperature=torch.zeros(1)), ValueError),
    (dict(logits=torch.zeros(2, 393217)), RuntimeError),
    (dict(logits=torch.zeros(2, 0)), RuntimeError),
    (dict(), RuntimeError),                         # host memory
])
def test_refusals(change, exc):
    H.ensure_built()
    a = dict(logits=torch.zeros(2, 8), out=torch.zeros(2, dtype=torch.int32), u=torch.zeros(2))
    a.update(change)
    with pytest.raises(exc):
        sample_rows(**a)


def test_plain_definition_by_hand():
    x = np.log(np.array([1, 4, 2, 1], np.float32))
    assert [plain(x, u, 1.0, 0, 1.0, 0.0) for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.9)] == [1, 1, 2, 2, 0, 3]
    assert [plain(x, u, 1.0, 2, 1.0, 0.0) for u in (0.0, 0.66, 0.67, 1.0)] == [1, 1, 2, 2]
    assert plain(x, 0.99, 1.0, 0, 0.5, 0.0) == 1 and plain(x, 0.99, 1.0, 0, 0.51, 0.0) == 2
    assert plain(x, 0.99, 1.0, 0, 1.0, 0.4) == 2 and plain(x, 0.9, 0.0, 0, 1.0, 0.0) == 1


# ---------------------------------------------------------------------- GPU ----

VOCABS = [1, 2, 3, 31, 32, 33, 640, 1000, 4097, 32000, 49152]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
                                dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.02),
                                dict(temperature=3.0, top_p=0.999), dict(top_k=10 ** 9, top_p=1e-9)])
def test_draws(dtype, vocab, kw):
    n = 24 if vocab < 10000 else 7
    draw(logits(n, vocab, vocab, dtype), us(n, vocab), **kw)


@pytest.mark.gpu
def test_mixed_rows_of_the_large_vocabulary():
    n = 16
    rng = np.random.default_rng(5)
    x = logits(n, 151936, 3)
    x[:8] += 8 * torch.rand(8, 151936, generator=torch.Generator().manual_seed(1)).cuda() ** 20
    draw(x, us(n), rng.uniform(0.3, 1.6, n), rng.integers(0, 2000, n) * (rng.random(n) < 0.5),
         np.where(rng.random(n) < 0.5, 1.0, rng.uniform(0.1, 0.99, n)), np.where(rng.random(n) < 0.5, 0.0, 0.01))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("scale", [0.3, 2.3])
def test_full_batches_next_to_borders(seed, scale):
    """thousands of untruncated draws: a weight that is off by 1e-8 of itself, or two
    neighbouring logits taken for one, changes one of them"""
    n, vocab = 256, 151936
    x = logits(n, vocab, seed, scale=scale)
    u, t = us(n, seed), np.random.default_rng(seed).uniform(0.5, 1.5, n).astype(np.float32)
    out = torch.empty(n, dtype=torch.int32, device="cuda")
    sample_rows(x, out, torch.tensor(u).cuda(), temperature=torch.tensor(t).cuda())
    l, index = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((l.double() - l[:, :1].double()) / torch.tensor(t).cuda()[:, None].double())
    run = torch.cumsum(w, -1)
    at = (run <= torch.tensor(u).cuda()[:, None].double() * run[:, -1:]).sum(-1, keepdim=True)
    assert torch.equal(out.long(), torch.gather(index, -1, at)[:, 0])


@pytest.mark.gpu
def test_largest_vocabulary():
    draw(logits(2, 393216, 1), us(2), top_p=0.9)
    draw(logits(2, 393216, 1, torch.float16), us(2))


PLANTED = {
    "flat": lambda x: x.zero_(),
    "ties": lambda x: x.copy_(torch.round(x)),
    "two values": lambda x: x.copy_(torch.where(x > 0, 1.0, 1.5)),
    "one dominant": lambda x: x.__setitem__((slice(None), 77), 300.0),
    "underflow": lambda x: x.mul_(200),
    "minus infinity": lambda x: x.masked_fill_(x < 0.5, -torch.inf),
    "nan": lambda x: x.masked_fill_(x > 2, torch.nan),
    "nan first": lambda x: x.__setitem__((slice(None), 0), torch.nan),
    "plus infinity": lambda x: x.__setitem__((slice(None), slice(5, 500, 7)), torch.inf),
    "all minus infinity": lambda x: x.fill_(-torch.inf),
    "all nan": lambda x: x.fill_(torch.nan),
    "all but one": lambda x: (x.fill_(-torch.inf), x.__setitem__((slice(None), 555), -3.0)),
    "zeros of both signs": lambda x: x.copy_(torch.where(x > 0, 0.0, -0.0)),
    "subnormal": lambda x: x.mul_(1e-39),
    "huge": lambda x: x.mul_(1e38),
    "steep cluster": lambda x: x.copy_(torch.where(x > -9, 5.0 + x * 1e-6, x)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [640, 20011])
@pytest.mark.parametrize("plant", sorted(PLANTED))
@pytest.mark.parametrize("kw", [dict(), dict(top_k=100, top_p=0.5), dict(min_p=0.5), dict(top_p=0.25), dict(temperature=0.0)])
def test_planted_rows(vocab, plant, kw):
    x = logits(9, vocab, 9)
    PLANTED[plant](x)
    draw(x, us(9, 4), **kw)


@pytest.mark.gpu
def test_ends_of_the_settings():
    x = torch.round(logits(12, 1000, 2) * 4) / 4
    u = np.array([0, 1 - 2 ** -24, 1.0, 2.0, -1.0, np.nan, np.inf, -np.inf, 0.5, 2 ** -24, 1e-30, 0.25], np.float32)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.3)):
        draw(x, u, **kw)
    t = np.array([1e-30, 1e30, np.inf, np.nan, -1, 1e-3, 1, 1, 1, 1, 1, 1], np.float32)
    draw(x, us(12), temperature=t)
    draw(x, us(12), top_k=np.array([-5, 0, 1, 2, 999, 1000, 1001, 2 ** 31 - 1, -2 ** 31, 5, 6, 7]))
    draw(x, us(12), top_p=np.array([0, -1, 1, 2, np.nan, 1e-12, 1 - 2 ** -24, 0.5, np.inf, 1e-45, 0.1, 0.9], np.float32))
    draw(x, us(12), min_p=np.array([0, -1, 1, 2, np.nan, 1e-12, 1 - 2 ** -24, 0.5, np.inf, 1e-45, 0.1, 0.9], np.float32))


@pytest.mark.gpu
def test_strides_alignment_and_neighbours():
    """odd strides and offsets give the aligned rows' tokens; the logits stay"""
    x = logits(6, 5003, 8)
    u, kw = us(6), dict(temperature=0.8, top_p=0.9)
    want = draw(x, u, **kw)
    for off, stride in ((0, 5003), (1, 5007), (3, 6001)):
        wide = torch.full((6, stride + 8), 1e9, device="cuda")
        view = wide[:, off:off + 5003]
        view.copy_(x)
        assert draw(view, u, **kw).tolist() == want.tolist()
        assert torch.equal(view, x) and (wide[:, off + 5003:] == 1e9).all()
    assert draw(x[2:3], u[2:3], **kw)[0] == want[2]
    same = x[:1].expand(6, 5003)                       # stride 0: one row of logits, six draws
    draw(same, u, **kw)


@pytest.mark.gpu
def test_stream_and_graph():
    x, n = logits(5, 32000, 4), 5
    u = torch.tensor(us(n)).cuda()
    p = torch.full((n,), 0.9, device="cuda")
    ref = torch.empty(n, dtype=torch.int32, device="cuda")
    sample_rows(x, ref, u, top_p=p)
    out = torch.zeros_like(ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sample_rows(x, out, u, top_p=p, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sample_rows(x, out, u, top_p=p, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        u.copy_(torch.rand(n, device="cuda"))
        g.replay()
        sample_rows(x, ref, u, top_p=p)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


@pytest.mark.gpu
def test_frequencies_of_a_known_distribution():
    """draws at evenly spaced u follow the weights exactly: token i's share of the
    grid differs from its probability by at most one grid step"""
    prob = np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    m = 4096
    x = torch.tensor(np.log(prob), dtype=torch.float32).cuda()[None].expand(m, 5)
    out = torch.empty(m, dtype=torch.int32, device="cuda")
    sample_rows(x, out, ((torch.arange(m) + 0.5) / m).cuda())
    share = np.bincount(out.cpu().numpy(), minlength=5) / m
    assert np.abs(share - prob).max() <= 1.0 / m
