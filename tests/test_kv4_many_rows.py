"""Every form of the many-row attention over the paged 4-bit cache (three head sizes,
two types, one or two row tiles a CTA) where it can go wrong: windows and sinks,
pages that are none, bytes never written, queries that are no numbers or far outside
fp16's range, rows that see nothing, strides, streams, graphs, pages behind 4 GiB.
Each test asks which kernel its sizes take, so that a change of that rule cannot
empty it."""
import ctypes

import numpy as np
import pytest

from emberllm_b200 import Ember, EmberBatch, Kv4Cache, synth

from . import helpers as H
from .test_kv4 import Paged, bound, plain_attention, plain_values

torch = pytest.importorskip("torch")
FEW_4, FEW_8, MANY_1, MANY_2 = 1, 2, 3, 4
F32, F16 = torch.float32, torch.float16


def kernel(dtype, max_q, heads, kvh, hd, seqs, tokens=None):
    hooks = H.testhooks()
    return hooks.ember_testhook_kv4_kernel(4 if dtype == F32 else 2, hd, tokens or seqs * max_q, max_q, heads // kvh, kvh,
                                           seqs)


# heads, kv heads, head_dim, rows a sequence at most, sequences; the kernel they take (fp16 heads of 32: one
# row tile always)
SHAPES = {
    "128-1": (16, 8, 128, 108, 3, MANY_1), "64-1": (14, 2, 64, 126, 3, MANY_1), "32-1": (9, 3, 32, 192, 3, MANY_1),
    "128-2": (16, 8, 128, 400, 3, MANY_2), "64-2": (14, 2, 64, 580, 6, MANY_2), "32-2": (16, 8, 32, 520, 6, MANY_2),
}
ALL = [pytest.param(s, d, id=f"{s}-{'f32' if d == F32 else 'f16'}") for s in SHAPES for d in (F32, F16)]


def make(shape, dtype, fill=0xAB, page=32, more=(3, 250, 0, 1000, 64, 17), short=(0, 7, 1, 0, 33, 2)):
    """ragged sequences of that shape: some rows and positions fewer or more each"""
    heads, kvh, hd, ql, seqs, want = SHAPES[shape]
    q = [ql - short[i] for i in range(seqs)]
    assert kernel(dtype, ql, heads, kvh, hd, seqs, sum(q)) == (MANY_1 if hd == 32 and dtype == F16 else want)
    p = Paged([n + more[i] for i, n in enumerate(q)], q, page, kvh, hd, seed=hd + ql, fill=fill)
    p.store_all()
    assert max(p.ql) == ql
    x = (torch.randn(sum(q), heads, hd, generator=torch.Generator().manual_seed(ql)) * 1.2).to(dtype).cuda()
    return p, x


def near(got, want):
    """fp32: sums cut at 24 bits and operands in 22 (derived in test_kv4_prompts.py);
    fp16: rounded once"""
    assert torch.isfinite(got).all()
    err = (got.double() - want).norm() / want.norm()
    if got.dtype == F32:
        assert err < 4e-6
    else:
        assert err < 1.02 * (want.half().double() - want).norm() / want.norm() + 5e-6


def test_which_kernel():
    """what the rule's comment says of the measured sizes"""
    k = lambda *a: kernel(F32, *a)
    assert k(1, 16, 8, 128, 64) == FEW_4 and k(1, 14, 2, 64, 512) == FEW_8 and k(256, 16, 8, 128, 1) == FEW_8
    assert k(32, 16, 8, 128, 8) == FEW_8 and k(64, 16, 8, 128, 8) == MANY_1 and k(32, 16, 8, 128, 64) == MANY_1
    assert k(512, 16, 8, 128, 1) == MANY_1 and k(512, 16, 8, 128, 4) == MANY_2 and k(4000, 16, 8, 128, 1) == MANY_2
    assert kernel(F16, 512, 16, 8, 128, 1) == MANY_2 and kernel(F16, 512, 14, 2, 64, 2) == MANY_1
    # a prompt among single tokens, ragged prompts, grids that would be empty or too large
    assert k(2000, 16, 8, 128, 201, 2200) >= MANY_1 and k(200000, 8, 8, 128, 4096, 237000) >= MANY_1
    assert k(4000, 16, 8, 128, 65535, 70000) >= MANY_1 and k(1, 16, 8, 128, 65535) == FEW_4
    assert k(256, 16, 8, 128, 64, 319) == FEW_8 and k(512, 16, 8, 128, 6, 1500) == MANY_2
    assert kernel(F16, 2000, 8, 1, 32, 8) == MANY_1 and k(2000, 8, 1, 32, 8) == MANY_2


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
@pytest.mark.parametrize("page", [16, 128])
def test_plain(shape, dtype, page):
    p, q = make(shape, dtype, page=page)
    near(p.attend(q), p.want(q))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (100, 19), (130, 300), (500, 500), (10000, 3)])
def test_windows_and_sinks(shape, dtype, window, sinks):
    p, q = make(shape, dtype)
    near(p.attend(q, window, sinks), p.want(q, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_pages_that_are_none(shape, dtype, window, sinks):
    """holes at the start, in the middle and behind the window; a sequence without any
    page; one without positions; rows before position 0"""
    p, q = make(shape, dtype)
    n0, ql = p.kv[1], p.ql
    p.table[1, 0], p.table[1, 3], p.table[1, 4] = -1, 2 ** 31 - 1, p.n_pages
    p.table[2] = -7
    lens = p.kv_len.clone()
    lens[0] = ql[0] - 20                                # its first 20 rows are before position 0
    if len(ql) > 3:
        lens[3] = 0
    out = torch.full_like(q, 5.0)
    p.cache.attention(q, out, p.start, lens, p.table, max(ql), max(p.kv), None, window, sinks, p.workspace(q.shape[1]))
    starts = np.cumsum([0] + ql)
    assert (out[:20] == 0).all() and (out[starts[2]:starts[3]] == 0).all()
    if len(ql) > 3:
        assert (out[starts[3]:starts[4]] == 0).all()
    hidden = torch.zeros(n0, dtype=torch.bool, device="cuda")
    hidden[0:32] = hidden[96:160] = True
    k, v = plain_values(p.k), plain_values(p.v)
    at = p.kv[0]
    pos = torch.arange(n0 - ql[1], n0, device="cuda")
    want = plain_attention(q[starts[1]:starts[2]].double(), k[at:at + n0], v[at:at + n0], pos, window, sinks,
                           p.hd ** -0.5, hidden)
    near(out[starts[1]:starts[2]], want)
    n = ql[0] - 20
    near(out[20:ql[0]], plain_attention(q[20:ql[0]].double(), k[:n], v[:n], torch.arange(n, device="cuda"), window, sinks,
                                        p.hd ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
def test_bytes_never_written_and_queries_that_are_no_numbers(shape, dtype):
    """unwritten scales are NaN here; a NaN or an infinity in a query stays in its row
    and head; rows of no sequence stay as they are"""
    p, q = make(shape, dtype, fill=0xFF, page=128)
    q = torch.cat([q, q[:3]])
    clean = p.attend(q)
    n = sum(p.ql)
    assert (clean[n:] == 77).all()
    near(clean[:n], p.want(q[:n]))
    bad = [(0, 0, torch.nan), (1, 2, torch.inf), (40, 1, -torch.inf), (n - 1, q.shape[1] - 1, torch.nan)]
    same = torch.ones(q.shape[:2], dtype=torch.bool)
    for row, head, value in bad:
        q[row, head, 3] = value
        same[row, head] = False
    got = p.attend(q)
    for row, head, _ in bad:
        assert torch.isnan(got[row, head]).all()
    assert torch.equal(got[same.cuda()], clean[same.cuda()])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("factor", [1e-38, 1e-30, 1e-6, 1e5, 1e20, 1e36])
def test_query_ranges(shape, factor):
    """queries far outside fp16's range, subnormal ones among them, the scale bringing
    the scores back (120 * 1e36 passes fp32's largest number in places: an infinite
    query's output is NaN)"""
    p, q = make(shape, F32)
    q[:, 0, 7] *= 100
    q = q * factor
    scale = float(np.float32(0.125 / factor)) if factor > 1e-30 else 1e29
    fine = torch.isfinite(q).all(-1)
    assert fine.all() or factor == 1e36
    smax = scale * q[fine].double().abs().sum(-1).amax().item() * 8
    got, want = p.attend(q, scale=scale), p.want(q, scale=scale)
    assert torch.isfinite(got[fine]).all() and torch.isnan(got[~fine]).all()
    assert (got.double() - want)[fine].abs().amax() <= bound(q, 8.0, smax, max(p.kv), F32)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
@pytest.mark.parametrize("scale", [-0.11, 0.0, 1e-30, 2.0])
def test_scales(shape, dtype, scale):
    """of either sign, none, and scores up to hundreds (weights of one position)"""
    p, q = make(shape, dtype)
    got, want = p.attend(q, scale=scale), p.want(q, scale=scale)
    if abs(scale) < 1:
        near(got, want)
    else:
        smax = scale * q.double().abs().sum(-1).amax().item() * 8
        assert (got.double() - want).abs().amax() <= bound(q, 8.0, smax, max(p.kv), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
@pytest.mark.parametrize("factor", [1e-5, 1000.0])
def test_value_ranges(shape, dtype, factor):
    """values among fp16's smallest and largest numbers"""
    p, q = make(shape, dtype)
    p.v *= factor
    p.store_all()
    got, want = p.attend(q), p.want(q)
    if dtype == F16 and factor < 1:
        # outputs among fp16's subnormal numbers, 2^-24 apart
        assert (got.double() - want).abs().amax() <= 2.0 ** -24
    else:
        near(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
def test_strides_and_tensors_beside(shape, dtype):
    p, q = make(shape, dtype)
    n, heads, hd = q.shape
    first = p.attend(q)
    wide = torch.full((n, heads + 1, hd + 3), 3.0, dtype=dtype, device="cuda")
    q2 = wide[:, 1:, 3:]
    q2.copy_(q)
    for off, pad in ((0, 0), (8, 8), (1, 1), (2, 4)):       # 16-byte accesses, and numbers one by one
        box = torch.full((heads, n, hd + off + pad), 9.0, dtype=dtype, device="cuda")
        out = box[:, :, off:off + hd].transpose(0, 1)
        assert torch.equal(p.attend(q2, out=out), first)
        assert (box[:, :, :off] == 9).all() and (box[:, :, off + hd:] == 9).all()
    # queries as a transposed tensor, one head's rows shared by all
    one = torch.randn(1, heads, hd, generator=torch.Generator().manual_seed(3)).to(dtype).cuda().expand(n, heads, hd)
    near(p.attend(one, out=torch.empty_like(q)), p.want(one))
    assert torch.equal(p.attend(q, max_kv=max(p.kv) + 1000), first)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", ALL)
def test_streams_graphs_and_again(shape, dtype):
    """two streams at once, with a workspace each; a graph of store and attention,
    replayed over changed keys; many runs give the first one's bits"""
    p, q = make(shape, dtype)
    first = p.attend(q)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in streams]
    ws = [p.workspace(q.shape[1]) for _ in streams]
    args = (p.start, p.kv_len, p.table, max(p.ql), max(p.kv))
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s, o, w in zip(streams, outs, ws):
            p.cache.attention(q, o, *args, workspace=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    g = torch.cuda.CUDAGraph()
    out = torch.zeros_like(q)
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream().cuda_stream
        p.cache.store(p.k, p.v, p.full, p.kv_len, p.table, max(p.kv), stream=st)
        p.cache.attention(q, out, *args, workspace=ws[0], stream=st)
    for r in range(4):
        p.k.neg_()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, p.attend(q))
        assert torch.equal(out, first) == (r % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,ql", [(16, 330), (16, 1500), (24, 220)])
def test_pages_behind_4_gib(dtype, heads, ql):
    page, kvh, hd = 128, 8, 128
    assert kernel(dtype, ql, heads, kvh, hd, 1) == (MANY_2 if ql == 1500 else MANY_1)
    n_pages = (5 << 30) // Kv4Cache.nbytes(1, page, kvh, hd)
    buf = torch.empty(Kv4Cache.nbytes(n_pages, page, kvh, hd), dtype=torch.uint8, device="cuda")
    cache = Kv4Cache(buf, n_pages, page, kvh, hd)
    n = 1600
    pages = [n_pages - 1, 0, n_pages // 2 + 7] + [n_pages - 2 - 3 * i for i in range(10)]
    table = torch.tensor([pages], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(n, kvh, hd, generator=g).cuda() for _ in range(2))
    lens, full = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([n], [0, n]))
    cache.store(k, v, full, lens, table, n)
    q = torch.randn(ql, heads, hd, generator=g).to(dtype).cuda()
    out = torch.empty_like(q)
    start = torch.tensor([0, ql], dtype=torch.int32).cuda()
    ws = torch.empty(max(16, cache.attention_workspace(heads, 1, ql, n)), dtype=torch.uint8, device="cuda")
    cache.attention(q, out, start, lens, table, ql, n, workspace=ws)
    near(out, plain_attention(q.double(), plain_values(k), plain_values(v), torch.arange(n - ql, n, device="cuda"), 0, 0,
                              hd ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("kv,ql,heads,kvh,hd,seqs", [(700, 1, 16, 8, 128, 1), (20011, 1, 16, 8, 128, 2), (2000, 1, 14, 2, 64, 90),
                                                     (5000, 2, 14, 2, 64, 3), (1200, 40, 12, 12, 64, 1), (40000, 3, 8, 1, 32, 1)])
def test_few_rows_are_as_exact(kv, ql, heads, kvh, hd, seqs):
    """the other kernel's sums are rounded: operands of 22 bits, scores of a few units
    and exponentials at 2^-22: below 1.5e-6 of the outputs at any length"""
    assert kernel(F32, ql, heads, kvh, hd, seqs) in (FEW_4, FEW_8)
    p = Paged([kv - 13 * i for i in range(seqs)], [ql] * seqs, 64, kvh, hd, seed=hd)
    p.store_all()
    q = (torch.randn(ql * seqs, heads, hd, generator=torch.Generator().manual_seed(2)) * 1.2).cuda()
    got, want = p.attend(q), p.want(q)
    assert (got.double() - want).norm() / want.norm() < 1.5e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,kvh,hd", [(16, 8, 128), (9, 3, 64)])
def test_prompts_among_single_tokens(dtype, heads, kvh, hd):
    """a step of many streams in which some start: both kernels take such batches"""
    for ql, want in (([1] * 20 + [256] + [1] * 20 + [0, 3], (FEW_8,)), ([1] * 5 + [600, 700, 1, 800], (MANY_1, MANY_2))):
        kv = [n + (97 * i) % 1500 for i, n in enumerate(ql)]
        p = Paged(kv, ql, 64, kvh, hd, seed=3)
        p.store_all()
        q = (torch.randn(sum(ql), heads, hd, generator=torch.Generator().manual_seed(2)) * 1.2).to(dtype).cuda()
        assert kernel(dtype, max(ql), heads, kvh, hd, len(ql), sum(ql)) in want
        near(p.attend(q), p.want(q))


# ---- the framework's own prompts in it ----

@pytest.mark.gpu
def test_a_streams_prompt_of_several_chunks(monkeypatch):
    """Chunks of 512 rows of one sequence take the many-row kernel, single tokens the
    other; both see the same cache but for a 4-bit or 8-bit code in 10^4 that falls
    the other way, so the logits point the same way."""
    assert kernel(F32, 512, 16, 8, 64, 1) == MANY_1 and kernel(F32, 1, 16, 8, 64, 2) == FEW_4
    monkeypatch.setitem(synth.CONFIGS, "tiny-heads", dict(
        dim=256, hidden_dim=512, n_layers=2, n_heads=16, n_kv_heads=8, head_dim=64, vocab_size=512, max_seq_len=2048,
        rope_theta=1e6, norm_eps=1e-6, rope_style=synth.ROPE_NEOX, tied=True, qk_norm=True, bias=False, quant="q8_0"))
    H.ensure_built()
    e = Ember(synth.ensure_model("tiny-heads"))
    ids = [int(t) for t in np.random.default_rng(1).integers(0, 512, 1400)]
    for kw in (dict(), dict(window=300, sinks=4)):
        b = EmberBatch(e, 2, max_steps=1, kv4=True, **kw)
        b.prefill(0, ids)                                # 512 + 512 + 376 rows
        b.prefill(1, ids[:600])
        for t in range(600, 1400):                       # the rest of it as single tokens
            b.greedy([7, ids[t]], [1400, t], 1)
        _, lg = b.greedy([7, 7], [1400, 1400], 1, logits=True)
        x = np.ctypeslib.as_array(lg).reshape(2, 512).astype(np.float64)
        assert np.isfinite(x).all()
        assert (x[0] * x[1]).sum() / np.linalg.norm(x[0]) / np.linalg.norm(x[1]) > 0.999
        b.close()
    e.close()
