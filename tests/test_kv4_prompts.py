"""Attention of many rows over the paged 4-bit cache: how exact its sums are, beyond
the worst-case bounds of test_kv4.py."""
import pytest

from .test_kv4 import Paged
from .test_kv4_many_rows import MANY_1, kernel

torch = pytest.importorskip("torch")


def queries(n, heads, hd, seed=1, scale=1.2, dtype=torch.float32):
    return (torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kvh,hd,seqs", [(16, 8, 128, 2), (16, 8, 128, 1), (12, 12, 64, 2), (9, 3, 64, 1), (8, 1, 32, 3)])
def test_half_precision_outputs_are_rounded_once(heads, kvh, hd, seqs):
    """fp16 outputs are the exact ones rounded, but for those next to a border of two
    numbers. Before that rounding an output is off by r of itself: the scores' products
    (at most 8 cuts at 24 bits of sums of a few units: 2e-6), the weights in 22 bits
    (2.4e-7), their sums over 900 positions (2.3e-9 each: 2e-6), which is less than
    r = 2e-5. An output moves across a border of numbers 2^-11 apart with the chance
    r / 2^-11, three times that for the small ones among them: 3 %. (Weights of 11 bits
    move 40 % of the outputs.)"""
    assert kernel(torch.float16, 900, heads, kvh, hd, seqs) >= MANY_1
    p = Paged([900 - 7 * i for i in range(seqs)], [900 - 7 * i for i in range(seqs)], 64, kvh, hd, seed=hd)
    p.store_all()
    q = queries(sum(p.ql), heads, hd, dtype=torch.float16)
    got, want = p.attend(q), p.want(q)
    once = want.half()
    assert (got != once).double().mean().item() < 0.03
    assert relative(got, want) < 1.01 * relative(once, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,ql,heads,kvh,hd,window,sinks", [
    ([1200, 700], [1200, 700], 16, 8, 128, 0, 0),
    ([20000], [330], 16, 8, 128, 0, 0), ([41000], [330], 16, 8, 128, 0, 0),
    ([3001], [3001], 12, 12, 64, 0, 0), ([9000, 520], [1300, 513], 9, 3, 64, 0, 0), ([6000] * 3, [400] * 3, 8, 1, 32, 0, 0),
    ([9000], [330], 16, 8, 128, 5000, 700)])
def test_single_precision_sums_at_any_length(kv, ql, heads, kvh, hd, window, sinks):
    """The tensor cores cut a running sum at 24 bits, twice for 16 positions: 64 times
    before it leaves them, half of 2^-23 of a sum that is on the average 2/3 of the
    segment's: 2.5e-6. The scores' own cuts (16 of sums of a few units, of both
    signs), 22 bits of queries and weights and the exponentials add less than 1.5e-6.
    (Sums that stay are off by 4.8e-5 at 20,000 positions.)"""
    assert kernel(torch.float32, max(ql), heads, kvh, hd, len(kv), sum(ql)) >= MANY_1
    p = Paged(kv, ql, 64, kvh, hd, seed=hd)
    p.store_all()
    q = queries(sum(ql), heads, hd)
    got, want = p.attend(q, window, sinks), p.want(q, window, sinks)
    assert relative(got, want) < 4e-6
    # the partial sums lie in the outputs' rows: strides, offsets and what is beside them
    n = sum(ql)
    wide = torch.full((heads + 1, n, hd + 3), 5.0, device="cuda")
    out = wide[1:, :, 3:].transpose(0, 1)
    p.attend(q, window, sinks, out=out)
    assert torch.equal(out, got) and (wide[0] == 5).all() and (wide[:, :, :3] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("kv,ql,heads,kvh,hd", [([6000] * 3, [400] * 3, 8, 1, 32), ([9000], [1300], 9, 3, 64), ([20000], [330], 16, 8, 128),
                                                ([3001], [3001], 12, 12, 64), ([4000, 2500], [900, 2500], 16, 8, 128)])
def test_long_ranges_again_and_again(dtype, kv, ql, heads, kvh, hd):
    """many runs give the first one's bits where sums leave tensor memory many times"""
    assert kernel(dtype, max(ql), heads, kvh, hd, len(kv), sum(ql)) >= MANY_1
    p = Paged(kv, ql, 64, kvh, hd, seed=hd)
    p.store_all()
    q = queries(sum(ql), heads, hd, dtype=dtype)
    first = p.attend(q)
    assert relative(first, p.want(q)) < (4e-6 if dtype == torch.float32 else 2.5e-4)
    for _ in range(60):
        assert torch.equal(p.attend(q), first)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,ql,heads,kvh,hd", [([6000] * 3, [400] * 3, 8, 1, 32), ([9000], [1301], 9, 3, 64), ([5000], [350], 16, 8, 128),
                                                ([3001], [3001], 12, 12, 64), ([4000, 2500], [900, 2500], 16, 8, 128)])
def test_sums_under_a_maximum_that_rises(kv, ql, heads, kvh, hd):
    """Scores from -25 to 25 along the sequence: the running maximum is raised some nine
    times, between the times at which the sums leave tensor memory and at them. A score's
    sum is cut 16 times and has 22 bits of its query: off by 25 * 20 * 2^-24 = 3e-5 at
    most, numerator and denominator twice that."""
    assert kernel(torch.float32, max(ql), heads, kvh, hd, len(kv), sum(ql)) >= MANY_1
    p = Paged(kv, ql, 64, kvh, hd, seed=hd)
    at = 0
    for n in kv:
        p.k[at:at + n, :, :32] = torch.linspace(-1, 1, n, device="cuda")[:, None, None]
        at += n
    p.store_all()
    q = queries(sum(ql), heads, hd, scale=0.5)
    q[..., :32] = 25 / 32 * hd ** 0.5
    got = p.attend(q)
    assert relative(got, p.want(q)) < 6e-5
    assert torch.equal(p.attend(q), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("kv,ql,heads,kvh,hd", [([2000, 700], [330, 600], 16, 8, 128), ([9000], [1301], 9, 3, 64), ([3000] * 4, [1] * 4, 16, 8, 128),
                                                ([20000], [5], 14, 2, 64)])
def test_outputs_in_place_of_the_queries(dtype, kv, ql, heads, kvh, hd):
    p = Paged(kv, ql, 64, kvh, hd, seed=hd)
    p.store_all()
    q = queries(sum(ql), heads, hd, dtype=dtype)
    want = p.attend(q)
    p.attend(q, out=q)
    assert torch.equal(q, want)
