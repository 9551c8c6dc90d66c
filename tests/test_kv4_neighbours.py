"""A row's attention over the paged 4-bit cache does not depend on its neighbours: the
other rows' and heads' queries may be anything, its bits stay; so may the bytes of
positions that no row sees."""
import pytest

from .test_kv4 import Paged
from .test_kv4_many_rows import MANY_1, kernel

torch = pytest.importorskip("torch")


def climbing(p, heads, seed):
    """queries whose scores rise along the sequence, each by its own slope: the
    running maximum passes the last one again and again"""
    g = torch.Generator().manual_seed(seed)
    slope = torch.rand(sum(p.ql), heads, 1, generator=g) * 60
    q = torch.randn(sum(p.ql), heads, p.hd, generator=g)
    q[..., :32] = slope
    return q


def ramp(p):
    """keys whose first block grows with the position"""
    at = 0
    for n in p.kv:
        p.k[at:at + n, :, :32] = torch.linspace(-1, 1, max(n, 1), device="cuda")[:n, None, None]
        at += n
    p.store_all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("kv,ql,heads,kvh,hd", [
    ([700, 150], [1, 1], 16, 8, 128), ([600, 90], [3, 2], 14, 2, 64),                      # few rows
    ([700, 520], [700, 520], 16, 8, 128), ([900], [900], 9, 3, 64), ([640] * 3, [400] * 3, 8, 1, 32),   # many
    ([500], [330], 16, 8, 128)])
def test_other_rows_queries_change_nothing(dtype, kv, ql, heads, kvh, hd):
    assert (kernel(dtype, max(ql), heads, kvh, hd, len(kv), sum(ql)) >= MANY_1) == (max(ql) > 3)
    p = Paged(kv, ql, 32, kvh, hd, seed=1)
    ramp(p)
    n = sum(ql)
    plain = (torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(5)) * 1.2).to(dtype)
    rise = climbing(p, heads, 6).to(dtype)
    first = p.attend(plain.cuda())
    # every second (row, head) climbs, then the others
    odd = (torch.arange(n)[:, None] + torch.arange(heads)[None]) % 2 == 1
    for mine in (odd, ~odd):
        q = torch.where(mine[..., None], rise, plain).cuda()
        got = p.attend(q)
        keep = ~mine.cuda()
        assert torch.equal(got[keep], first[keep])
    # and the climbing ones among each other
    both = p.attend(rise.cuda())
    q = torch.where(odd[..., None], rise, rise.flip(0)).cuda()
    assert torch.equal(p.attend(q)[odd.cuda()], both[odd.cuda()])
    # (scores up to 60 * 32 * hd^-0.5 <= 340 in sums of hd products: weights off by
    # 2 * 340 * (hd + 8) * 2^-24 <= 5.6e-3, values below 8)
    want = p.want(rise.cuda())
    assert torch.isfinite(both).all() and (both.double() - want).abs().amax() < 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("window,sinks", [(100, 4), (33, 0), (250, 19), (1, 1), (700, 33), (64, 64)])
@pytest.mark.parametrize("kv,ql,heads,kvh,hd", [([1500, 811], [1, 1], 16, 8, 128), ([1500, 811], [3, 2], 14, 2, 64),
                                                ([1500, 811], [300, 130], 16, 8, 128), ([1000] * 6, [430] * 6, 9, 3, 32)])
def test_positions_that_nobody_sees_need_not_be_written(dtype, window, sinks, kv, ql, heads, kvh, hd):
    """a program that keeps the first tokens and a window writes nothing else: the
    other bytes are NaN scales here, in the same pages and groups"""
    assert (kernel(dtype, max(ql), heads, kvh, hd, len(kv), sum(ql)) >= MANY_1) == (max(ql) > 3)
    p = Paged(kv, ql, 64, kvh, hd, seed=window)
    p.store_all()
    q = (torch.randn(sum(ql), heads, hd, generator=torch.Generator().manual_seed(3)) * 1.2).to(dtype).cuda()
    want = p.attend(q, window, sinks)
    assert torch.isfinite(want).all()
    p.buf.fill_(0xFF)
    at = 0
    for i, (n, m) in enumerate(zip(kv, ql)):
        for end, rows in ((min(sinks, n), min(sinks, n)), (n, min(n, window + m - 1))):
            if rows:
                start = torch.tensor([0, rows], dtype=torch.int32).cuda()
                lens = torch.tensor([end], dtype=torch.int32).cuda()
                src = slice(at + end - rows, at + end)
                p.cache.store(p.k[src], p.v[src], start, lens, p.table[i:i + 1], rows)
        at += n
    assert torch.equal(p.attend(q, window, sinks), want)
