"""The paged 4-bit KV cache and the attention over it, against plain 64-bit
implementations of their definitions (include/ember_kv4.h)."""
import ctypes
import os
import re

import numpy as np
import pytest

from emberllm_b200 import Kv4Cache, _lib, kv4

from . import helpers as H

torch = pytest.importorskip("torch")
HDR = os.path.join(H.ROOT, "include", "ember_kv4.h")


# ------------------------------------------------------- plain definitions ----

def plain_blocks(x):
    """(codes, scales) of rows of 32-element blocks in float64"""
    x = torch.nan_to_num(x.float(), nan=0.0).double().unflatten(-1, (-1, 32))
    mag = x.abs()
    first = (mag == mag.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
    d = (torch.gather(x, -1, first) / -8).clamp(-8160, 8160).to(torch.bfloat16).half().double()
    code = torch.floor(x / torch.where(d == 0, 1.0, d) + 8.5).clamp(0, 15)
    return torch.where(d == 0, 8.0, code), d


def plain_values(x):
    code, d = plain_blocks(x)
    return ((code - 8) * d).flatten(-2)


def plain_attention(q, k, v, pos, window, sinks, scale, hidden=None):
    """q [rows][heads][hd] at positions pos, k and v [len][kv heads][hd], float64"""
    rows, heads, hd = q.shape
    kvh = k.shape[1]
    p = torch.arange(k.shape[0], device=q.device)
    see = p[None] <= pos[:, None]
    if window:
        see &= (pos[:, None] - p[None] < window) | (p[None] < sinks)
    if hidden is not None:
        see &= ~hidden[None]
    kk, vv = (t.repeat_interleave(heads // kvh, 1) for t in (k, v))
    s = torch.einsum("mhd,nhd->hmn", q, kk) * scale
    s = s.masked_fill(~see[None], -torch.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    e = torch.where(see[None], e, 0.0)
    z = e.sum(-1, keepdim=True)
    return torch.einsum("hmn,nhd->mhd", e / torch.where(z == 0, 1.0, z), vv)


class Paged:
    """ragged sequences in shuffled pages, with a few spare pages"""

    def __init__(self, kv, ql, page, kvh, hd, seed=0, dtype=torch.float32, fill=0xAB):
        self.kv, self.ql, self.page, self.kvh, self.hd = kv, ql, page, kvh, hd
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in kv]
        self.n_pages = sum(need) + 5
        order = torch.randperm(self.n_pages, generator=g).tolist()
        width = max(1, max(need))
        table = torch.full((len(kv), width), -1, dtype=torch.int32)
        for i, n in enumerate(need):
            table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.table = table.cuda()
        self.start = torch.tensor([0] + list(np.cumsum(ql)), dtype=torch.int32).cuda()
        self.full = torch.tensor([0] + list(np.cumsum(kv)), dtype=torch.int32).cuda()
        self.kv_len = torch.tensor(kv, dtype=torch.int32).cuda()
        n = Kv4Cache.nbytes(self.n_pages, page, kvh, hd)
        self.buf = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        self.cache = Kv4Cache(self.buf, self.n_pages, page, kvh, hd)
        self.k = torch.randn(sum(kv), kvh, hd, generator=g).to(dtype).cuda()
        self.v = torch.randn(sum(kv), kvh, hd, generator=g).to(dtype).cuda()

    def store_all(self):
        self.cache.store(self.k, self.v, self.full, self.kv_len, self.table, max(self.kv))

    def workspace(self, heads, max_q=None, max_kv=None):
        n = self.cache.attention_workspace(heads, len(self.kv), max_q or max(1, max(self.ql)), max_kv or max(1, max(self.kv)))
        return torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")

    def attend(self, q, window=0, sinks=0, scale=None, out=None, max_q=None, max_kv=None, **kw):
        out = torch.full_like(q, 77.0) if out is None else out
        ws = self.workspace(q.shape[1], max_q, max_kv)
        self.cache.attention(q, out, self.start, self.kv_len, self.table, max_q or max(1, max(self.ql)),
                             max_kv or max(1, max(self.kv)), scale, window, sinks, ws, **kw)
        return out

    def want(self, q, window=0, sinks=0, scale=None):
        res, at, kat = [], 0, 0
        for n, m in zip(self.kv, self.ql):
            k = plain_values(self.k[kat:kat + n]) if n else self.k[:0].double()
            v = plain_values(self.v[kat:kat + n]) if n else self.v[:0].double()
            pos = torch.arange(n - m, n, device="cuda")
            if n:
                res.append(plain_attention(q[at:at + m].double(), k, v, pos, window, sinks,
                                           self.hd ** -0.5 if scale is None else scale))
            else:
                res.append(torch.zeros(m, q.shape[1], self.hd, dtype=torch.float64, device="cuda"))
            at, kat = at + m, kat + n
        return torch.cat(res)


def bound(q, vmax, smax, n, dtype):
    """How far an output may be off. A score is a sum of head_dim products of the
    query in 22 bits with exact cache values, accumulated in fp32: at most
    (2^-22 + (head_dim + 8) * 2^-24) * sum |q k|, with smax a bound of scale *
    sum |q k|; exp turns that into a relative error of each weight, to which exp
    itself (2^-21 relative to scores of this size) and 22 bits of the weight add.
    The output is a mean of values below vmax: twice the relative error (numerator
    and denominator) times vmax, the fp32 accumulation of n terms (errors of
    rounding add in the square root: 8 * sqrt(n) * 2^-24 covers them), and half a
    step of the output's type (fp16 weights of many-row calls: 2^-11 more)."""
    hd = q.shape[-1]
    rel = smax * (2.0 ** -22 + (hd + 8) * 2.0 ** -24) + 2.0 ** -20 + 8 * n ** 0.5 * 2.0 ** -24
    half = 2.0 ** -11 + 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    return vmax * (2 * rel + half)


def check(p, q, window=0, sinks=0, scale=None):
    got = p.attend(q, window, sinks, scale)
    want = p.want(q, window, sinks, scale)
    kv = plain_values(p.k).abs().amax().item() if sum(p.kv) else 0.0
    vmax = plain_values(p.v).abs().amax().item() if sum(p.kv) else 0.0
    sc = p.hd ** -0.5 if scale is None else abs(scale)
    smax = sc * q.double().abs().sum(-1).amax().item() * kv
    err = (got.double() - want).abs().amax().item() if got.numel() else 0.0
    assert err <= bound(q, vmax, smax, max(p.kv), q.dtype), err
    return got


# ---------------------------------------------------------------------- CPU ----

def test_declared_functions_are_exported_and_listed():
    H.ensure_built()
    lib = _lib.load()
    text = re.sub(r"/\*.*?\*/", "", open(HDR).read(), flags=re.S)
    names = set(re.findall(r"\b(ember_\w+)\s*\(", text))
    assert names and names == set(_lib.KV4_SYMBOLS)
    assert all(hasattr(lib, n) for n in names)


def test_packed_structures_are_the_headers(tmp_path):
    """the Python face packs the header's structures itself: sizes and last fields"""
    import subprocess
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text("""#include "ember_kv4.h"
#include <stddef.h>
#include <stdio.h>
int main(void) { printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(EmberKv4Cache), sizeof(EmberKv4Batch),
    sizeof(EmberKv4Rows), sizeof(EmberKv4Attention), sizeof(EmberSampleRows), offsetof(EmberKv4Attention, workspace),
    offsetof(EmberSampleRows, stride)); }
""")
    subprocess.run(["gcc", "-I" + os.path.join(H.ROOT, "include"), "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert got == [s.size for s in (kv4._CACHE, kv4._BATCH, kv4._ROWS, kv4._ATT, kv4._SAMPLE)] + [72, 24]
    assert kv4._ATT.unpack(kv4._ATT.pack(1, 2, 3, 4, 5, 6, 7, 8, 0.5, 9, 10, 11, 12, 13))[-2:] == (12, 13)


@pytest.mark.parametrize("args", [(0, 16, 1, 64), (4, 24, 1, 64), (4, 8, 1, 64), (4, 256, 1, 64), (4, 16, 0, 64),
                                  (4, 16, 1, 96), (4, 16, 1, 256), (1 << 28, 16, 1, 64), (-1, 16, 1, 64)])
def test_cache_sizes_refused(args):
    H.ensure_built()
    assert _lib.load().ember_cuda_kv4_bytes(*args) == 0
    with pytest.raises(ValueError):
        Kv4Cache.nbytes(*args)


@pytest.mark.parametrize("page,kvh,hd", [(16, 1, 32), (64, 8, 128), (128, 2, 64)])
def test_cache_bytes(page, kvh, hd):
    H.ensure_built()
    # 4 bits an element and an fp16 scale per 32, keys and values
    assert Kv4Cache.nbytes(7, page, kvh, hd) == 7 * page * kvh * 2 * (hd // 2 + hd // 32 * 2)


def cpu_call(**change):
    """an attention call on host memory, which the checks refuse before any launch"""
    H.ensure_built()
    p = Paged.__new__(Paged)
    buf = torch.zeros(Kv4Cache.nbytes(4, 16, 2, 64) + 16, dtype=torch.uint8)
    cache = Kv4Cache(buf, 4, 16, 2, 64)
    if "cache" in change:
        c = dict(page_size=16, head_dim=64)
        c.update(change.pop("cache"))
        cache._p = kv4._CACHE.pack(buf.data_ptr(), 4, c["page_size"], 2, c["head_dim"])
    q = change.pop("q", torch.zeros(3, 4, 64))
    out = change.pop("out", torch.zeros_like(q))
    kw = dict(max_q=1, max_kv=16, window=0, sinks=0)
    kw.update(change)
    start = kw.pop("start", torch.tensor([0, 1, 2, 3], dtype=torch.int32))
    lens = kw.pop("lens", torch.tensor([1, 2, 3], dtype=torch.int32))
    table = kw.pop("table", torch.zeros(3, 1, dtype=torch.int32))
    cache.attention(q, out, start, lens, table, **kw)


@pytest.mark.parametrize("change,exc,msg", [
    (dict(q=torch.zeros(3, 4, 32)), ValueError, "must be"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), ValueError, "float32 or float16"),
    (dict(q=torch.zeros(3, 4, 128)[:, :, ::2]), ValueError, "consecutive"),
    (dict(out=torch.zeros(2, 4, 64)), ValueError, "same rows"),
    (dict(out=torch.zeros(3, 4, 64).half()), ValueError, "same rows"),
    (dict(start=torch.zeros(3, dtype=torch.int32)), ValueError, "q_start"),
    (dict(start=torch.zeros(4, dtype=torch.int64)), ValueError, "q_start"),
    (dict(table=torch.zeros(2, 1, dtype=torch.int32)), ValueError, "block_table"),
    (dict(table=torch.zeros(3, 4, dtype=torch.int32)[:, :2]), ValueError, "contiguous"),
    (dict(cache=dict(page_size=24)), RuntimeError, "not supported"),
    (dict(cache=dict(head_dim=96), q=torch.zeros(3, 4, 64)), RuntimeError, "not supported"),
    (dict(max_q=-1), RuntimeError, "max_q"),
    (dict(), RuntimeError, "device memory"),
])
def test_attention_refusals_on_the_host(change, exc, msg):
    with pytest.raises(exc, match=msg):
        cpu_call(**change)


def test_store_refusals_on_the_host():
    H.ensure_built()
    cache = Kv4Cache(torch.zeros(Kv4Cache.nbytes(4, 16, 2, 64), dtype=torch.uint8), 4, 16, 2, 64)
    lens, table = torch.tensor([1], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    k = torch.zeros(1, 2, 64)
    for kk, vv, exc in ((k, torch.zeros(2, 2, 64), ValueError), (k, k.half(), ValueError), (k[:, :1], k, ValueError),
                        (k.double(), k.double(), ValueError), (k, k, RuntimeError)):
        with pytest.raises(exc):
            cache.store(kk, vv, None, lens, table)
    with pytest.raises(ValueError):
        Kv4Cache(torch.zeros(100, dtype=torch.uint8), 4, 16, 2, 64)


# ---------------------------------------------------------------------- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd,kvh,page", [(32, 3, 16), (64, 2, 32), (128, 8, 64), (128, 1, 128)])
def test_store_and_read(dtype, hd, kvh, page):
    """cached values equal the definition exactly (whole steps and fp16 scales)"""
    p = Paged([1, 37, page, 3 * page + 1, 130], [1] * 5, page, kvh, hd, seed=hd, dtype=dtype)
    p.k[5] *= 1e-4
    p.k[6] *= 1e-7 if dtype == torch.float16 else 1e-9     # scales among fp16's smallest, or zero
    p.k[7] *= 6000
    p.k[8] = 0
    p.v[3, :, :32] = 5.0
    p.v[4, :, 1::2] *= -1
    p.v[4] = p.v[4].abs().amax() * torch.sign(p.v[4])       # ties of magnitude: the first decides
    if dtype == torch.float32:
        p.v[9] *= 1e30                                      # saturates
    p.store_all()
    kb, vb = torch.full_like(p.k, 7), torch.full_like(p.v, 7)
    p.cache.read(kb, vb, p.full, p.kv_len, p.table, max(p.kv))
    assert torch.equal(kb.double(), plain_values(p.k))
    assert torch.equal(vb.double(), plain_values(p.v))
    # what is read back stores to the same values
    p.cache.store(kb, vb, p.full, p.kv_len, p.table, max(p.kv))
    k2, v2 = torch.empty_like(kb), torch.empty_like(vb)
    p.cache.read(k2, v2, p.full, p.kv_len, p.table, max(p.kv))
    assert torch.equal(k2, kb) and torch.equal(v2, vb)


@pytest.mark.gpu
def test_store_codes_next_to_borders():
    """values half a step between two codes, and their fp32 neighbours"""
    p = Paged([512], [1], 16, 1, 32)
    g = torch.Generator().manual_seed(3)
    d = (torch.rand(512, 1, generator=g) * 3 + 0.01).bfloat16().float()
    border = (torch.randint(-7, 8, (512, 32), generator=g) + 0.5) * d
    step = torch.randint(-1, 2, (512, 32), generator=g)
    x = torch.where(step == 0, border, torch.nextafter(border, torch.where(step > 0, torch.inf, -torch.inf)))
    x[:, 0] = -8 * d[:, 0]
    p.k[:, 0] = x.cuda()
    p.v[:, 0] = -x.cuda()
    p.store_all()
    kb, vb = torch.empty_like(p.k), torch.empty_like(p.v)
    p.cache.read(kb, vb, p.full, p.kv_len, p.table, 512)
    assert torch.equal(kb.double(), plain_values(p.k)) and torch.equal(vb.double(), plain_values(p.v))


@pytest.mark.gpu
def test_store_of_what_is_no_number():
    p = Paged([40], [40], 16, 2, 64)
    p.k[3, 0, 5] = torch.nan
    p.k[4, 1, 63] = torch.inf
    p.v[5, 0] = torch.nan
    p.v[6, 1, 0] = -torch.inf
    p.store_all()
    kb, vb = torch.empty_like(p.k), torch.empty_like(p.v)
    p.cache.read(kb, vb, p.full, p.kv_len, p.table, 40)
    assert torch.isfinite(kb).all() and torch.isfinite(vb).all()
    assert torch.equal(kb.double(), plain_values(p.k)) and torch.equal(vb.double(), plain_values(p.v))
    assert kb[4, 1, 63] == 65280 and vb[6, 1, 0] == -65280


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["last rows", "strides", "no q_start", "bad pages", "behind the batch"])
def test_store_rows(case):
    """which slots a store writes; every other byte of the cache stays"""
    p = Paged([20, 0, 33, 16], [20, 0, 33, 16], 16, 2, 64, seed=1)
    p.store_all()
    before = p.buf.clone()
    g = torch.Generator().manual_seed(9)
    if case == "last rows":
        ql = [3, 0, 17, 1]
        start = torch.tensor([0, 3, 3, 20, 21], dtype=torch.int32).cuda()
        k, v = (torch.randn(21, 2, 64, generator=g).cuda() for _ in range(2))
        p.cache.store(k, v, start, p.kv_len, p.table, 17)
        at, kat = 0, 0
        for n, m in zip(p.kv, ql):
            p.k[kat + n - m:kat + n], p.v[kat + n - m:kat + n] = k[at:at + m], v[at:at + m]
            at, kat = at + m, kat + n
    elif case == "strides":
        k = torch.randn(2, 69, 70, generator=g).cuda()[:, :, 3:67].transpose(0, 1)
        v = torch.randn(69, 3, 64, generator=g).cuda()[:, 1:]
        p.cache.store(k, v, p.full, p.kv_len, p.table, 33)
        p.k, p.v = k.clone(), v.clone()
    elif case == "no q_start":
        k, v = (torch.randn(4, 2, 64, generator=g).cuda() for _ in range(2))
        p.cache.store(k, v, None, p.kv_len, p.table)
        for i, r in ((0, 19), (2, 52), (3, 68)):       # sequence 1 is empty: its row is not stored
            p.k[r], p.v[r] = k[i], v[i]
    elif case == "bad pages":
        bad = p.table.clone()
        bad[0, 0], bad[2, 1], bad[3, 0] = p.n_pages, -5, 2 ** 31 - 1
        k, v = (torch.randn(69, 2, 64, generator=g).cuda() for _ in range(2))
        p.cache.store(k, v, p.full, p.kv_len, bad, 33)
        keep = torch.ones(69, dtype=torch.bool)
        keep[0:16] = keep[36:52] = keep[53:69] = False
        p.k[keep.cuda()], p.v[keep.cuda()] = k[keep.cuda()], v[keep.cuda()]
    else:
        start = torch.tensor([0, 5, 5, 9, 2 ** 31 - 1], dtype=torch.int32).cuda()   # sequence 3: rows 9..11 of 12
        lens = torch.tensor([20, 0, 33, 2], dtype=torch.int32).cuda()               # its first row is at position -1
        k, v = (torch.randn(12, 2, 64, generator=g).cuda() for _ in range(2))
        p.cache.store(k, v, start, lens, p.table, 5)
        for rows, dst in ((slice(0, 5), slice(15, 20)), (slice(5, 9), slice(49, 53)), (slice(10, 12), slice(53, 55))):
            p.k[dst], p.v[dst] = k[rows], v[rows]
    got = p.buf.clone()
    p.buf.copy_(before)
    p.store_all()
    assert torch.equal(got, p.buf)


HEADS = [(16, 8, 128), (14, 2, 64), (9, 3, 64), (12, 12, 64), (8, 1, 32), (3, 1, 32), (40, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("heads,kvh,hd", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_attention_single_tokens(dtype, heads, kvh, hd, page):
    p = Paged([1, 2, 15, 16, 17, 63, 64, 65, 200, 777], [1] * 10, page, kvh, hd, seed=heads)
    p.store_all()
    q = (torch.randn(10, heads, hd, generator=torch.Generator().manual_seed(1)) * 1.5).to(dtype).cuda()
    got = check(p, q)
    # without q_start, and in other strides
    wide = torch.zeros(10, heads + 1, hd + 3, dtype=dtype, device="cuda")
    q2 = wide[:, 1:, 3:]
    q2.copy_(q)
    out = torch.zeros(heads, 10, hd, dtype=dtype, device="cuda").transpose(0, 1)
    p.cache.attention(q2, out, None, p.kv_len, p.table, max_kv=777, workspace=p.workspace(heads))
    assert torch.equal(out, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (100, 19), (500, 500), (10000, 3)])
@pytest.mark.parametrize("ql", [1, 3, 70])
def test_attention_window_and_sinks(dtype, window, sinks, ql):
    kv = [ql, ql + 1, 90, 400, 1203]
    p = Paged(kv, [ql] * 5, 32, 2, 64, seed=window)
    p.store_all()
    q = torch.randn(5 * ql, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    check(p, q, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("heads,kvh,hd", HEADS)
def test_attention_ragged_prompts(dtype, heads, kvh, hd):
    p = Paged([1, 130, 64, 300, 257, 5, 0, 129], [1, 130, 1, 100, 64, 2, 0, 129], 16, kvh, hd, seed=hd)
    p.store_all()
    q = torch.randn(sum(p.ql), heads, hd, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    check(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 2, 4, 5, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("heads,kvh", [(4, 4), (6, 2), (7, 1)])
def test_attention_few_tokens(ql, heads, kvh):
    p = Paged([ql, 100, 515], [ql] * 3, 16, kvh, 64, seed=ql)
    p.store_all()
    q = torch.randn(3 * ql, heads, 64, generator=torch.Generator().manual_seed(ql)).cuda()
    check(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("ql", [1, 40])
def test_attention_long(dtype, ql):
    p = Paged([20011, 333], [ql, ql], 64, 2, 128, seed=5)
    p.store_all()
    q = (torch.randn(2 * ql, 4, 128, generator=torch.Generator().manual_seed(6)) * 2).to(dtype).cuda()
    check(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 50])
@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1e5, 1e20])
def test_attention_query_ranges(ql, factor):
    """queries far outside fp16's range, the scale bringing the scores back"""
    p = Paged([120], [ql], 16, 2, 64, seed=8)
    p.store_all()
    q = torch.randn(ql, 4, 64, generator=torch.Generator().manual_seed(3)).cuda()
    q[:, 0, 7] *= 100
    check(p, q * factor, scale=float(np.float32(0.125 / factor)))


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 50])
@pytest.mark.parametrize("factor", [1e-5, 1000.0])
def test_attention_value_ranges(ql, factor):
    p = Paged([120], [ql], 16, 2, 64, seed=8)
    p.v *= factor
    p.store_all()
    check(p, torch.randn(ql, 4, 64, generator=torch.Generator().manual_seed(3)).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 2, 60])
def test_attention_rows_that_see_nothing(ql):
    """no positions at all, invalid pages, rows before position 0: zeros"""
    p = Paged([0, 100, 60, 100], [ql] * 4, 16, 2, 64, seed=2)
    p.store_all()
    p.table[1] = -1
    p.table[3, 0] = 2 ** 31 - 1                        # its first 16 positions are hidden
    lens = torch.tensor([0, 100, ql - 1, 100], dtype=torch.int32).cuda()
    q = torch.randn(4 * ql, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.full_like(q, 5.0)
    p.cache.attention(q, out, p.start, lens, p.table, ql, 100, workspace=p.workspace(4))
    assert (out[:2 * ql] == 0).all()
    assert (out[2 * ql] == 0).all()                    # sequence 2: position -1
    hidden = torch.arange(100, device="cuda") < 16
    k, v = plain_values(p.k[160:260]), plain_values(p.v[160:260])
    want = plain_attention(q[3 * ql:].double(), k, v, torch.arange(100 - ql, 100, device="cuda"), 0, 0, 0.125, hidden)
    assert (out[3 * ql:].double() - want).abs().amax() <= bound(q, 10.0, 60.0, 100, q.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 40])
def test_attention_looks_at_nothing_it_must_not(ql):
    """bytes that were never stored are NaN scales here; NaN queries stay in their
    own (row, head); rows of no sequence stay as they are"""
    p = Paged([45, 100, 17], [ql if ql == 1 else 17] * 3, 16, 2, 64, seed=4, fill=0xFF)
    p.store_all()
    m = p.ql[0]
    q = torch.randn(3 * m + 2, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    clean = p.attend(q)
    assert torch.isfinite(clean).all() and (clean[3 * m:] == 77).all()
    assert (clean[:3 * m].double() - p.want(q)).abs().amax() <= bound(q, 8.0, 60.0, 100, q.dtype)
    q[1, 2, 3] = torch.nan
    q[2, 0, 0] = torch.inf
    got = p.attend(q)
    assert torch.isnan(got[1, 2]).all() and torch.isnan(got[2, 0]).all()
    same = torch.ones(q.shape[:2], dtype=torch.bool)
    same[1, 2] = same[2, 0] = False
    assert torch.equal(got[same.cuda()], clean[same.cuda()])


@pytest.mark.gpu
@pytest.mark.parametrize("ql", [1, 50])
def test_attention_neighbours_streams_and_graphs(ql):
    """the same call gives the same bits: alone on another stream, and replayed"""
    p = Paged([300, 77, 1000], [ql] * 3, 32, 2, 64, seed=11)
    p.store_all()
    q = torch.randn(3 * ql, 6, 64, generator=torch.Generator().manual_seed(1)).cuda()
    first = p.attend(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out, ws = torch.zeros_like(q), p.workspace(6)
    args = (p.start, p.kv_len, p.table, ql, 1000)
    with torch.cuda.stream(s):
        p.cache.attention(q, out, *args, workspace=ws, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream().cuda_stream
        p.cache.store(p.k, p.v, p.full, p.kv_len, p.table, 1000, stream=st)
        p.cache.attention(q, out, *args, workspace=ws, stream=st)
    for r in range(3):
        p.k.neg_()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        ref = p.attend(q)
        assert torch.equal(out, ref)
        assert (torch.equal(ref, first)) == (r % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("heads,kvh,hd", [(12, 12, 64), (40, 2, 128), (16, 8, 128)])
def test_attention_prompts_again_and_again(dtype, heads, kvh, hd):
    """many runs give the first one's bits: no wait that sometimes passes early"""
    p = Paged([1, 130, 64, 300, 257, 5, 0, 129], [1, 130, 1, 100, 64, 2, 0, 129], 16, kvh, hd, seed=hd)
    p.store_all()
    q = torch.randn(sum(p.ql), heads, hd, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    first = check(p, q)
    for _ in range(40):
        assert torch.equal(p.attend(q), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("seqs,ql,heads,kvh,hd", [(1, 40, 16, 8, 128), (40, 40, 16, 8, 128), (40, 33, 9, 3, 64),
                                                  (2, 700, 4, 2, 64), (3, 600, 8, 1, 32), (70, 9, 16, 8, 128)])
def test_attention_between_few_and_many_rows(dtype, seqs, ql, heads, kvh, hd):
    """both kernels, in contiguous tensors and in odd strides and offsets"""
    kv = [ql + (37 * i) % 300 for i in range(seqs)]
    p = Paged(kv, [ql - i % min(ql, 7) for i in range(seqs)], 32, kvh, hd, seed=ql)
    p.store_all()
    n = sum(p.ql)
    q = torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(ql)).to(dtype).cuda()
    got = check(p, q)
    wide = torch.zeros(n, heads + 1, hd + 3, dtype=dtype, device="cuda")
    q2 = wide[:, 1:, 3:]
    q2.copy_(q)
    out = torch.zeros(heads, n, hd + 1, dtype=dtype, device="cuda")[:, :, 1:].transpose(0, 1)
    assert torch.equal(p.attend(q2, out=out, max_q=ql), got)
    assert (wide[:, 0] == 0).all() and (wide[:, :, :3] == 0).all()


@pytest.mark.gpu
def test_attention_large_offsets():
    """a cache of more than 2^32 bytes: pages behind 4 GiB"""
    page, kvh, hd = 128, 8, 128
    n_pages = (5 << 30) // Kv4Cache.nbytes(1, page, kvh, hd)
    buf = torch.empty(Kv4Cache.nbytes(n_pages, page, kvh, hd), dtype=torch.uint8, device="cuda")
    cache = Kv4Cache(buf, n_pages, page, kvh, hd)
    table = torch.tensor([[n_pages - 1, 0, n_pages // 2 + 7]], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(300, kvh, hd, generator=g).cuda() for _ in range(2))
    lens = torch.tensor([300], dtype=torch.int32).cuda()
    full = torch.tensor([0, 300], dtype=torch.int32).cuda()
    cache.store(k, v, full, lens, table, 300)
    for ql in (1, 40):
        q = torch.randn(ql, 16, hd, generator=g).cuda()
        out = torch.empty_like(q)
        start = torch.tensor([0, ql], dtype=torch.int32).cuda()
        ws = torch.empty(max(16, cache.attention_workspace(16, 1, ql, 300)), dtype=torch.uint8, device="cuda")
        cache.attention(q, out, start, lens, table, ql, 300, workspace=ws)
        want = plain_attention(q.double(), plain_values(k), plain_values(v),
                               torch.arange(300 - ql, 300, device="cuda"), 0, 0, hd ** -0.5)
        assert (out.double() - want).abs().amax() <= bound(q, 8.0, 60.0, 300, q.dtype)


@pytest.mark.gpu
def test_attention_refusals_on_the_device():
    p = Paged([5000], [1], 16, 2, 64)
    q = torch.zeros(1, 4, 64, device="cuda")
    need = p.cache.attention_workspace(4, 1, 1, 5000)
    call = lambda **kw: p.cache.attention(q, torch.zeros_like(q), p.start, p.kv_len, p.table, **{**dict(max_kv=5000, workspace=p.workspace(4)), **kw})
    call()
    for kw, msg in ((dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(scale=float("nan")), "scale"),
                    (dict(max_kv=-1), "max_kv")):
        with pytest.raises(RuntimeError, match=msg):
            call(**kw)
    if need:
        with pytest.raises(RuntimeError, match="workspace"):
            call(workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
        with pytest.raises(RuntimeError, match="workspace"):
            call(workspace=torch.empty(need + 64, dtype=torch.uint8, device="cuda")[1:])
    with pytest.raises(RuntimeError, match="multiple"):
        p.cache.attention(q[:, :3], q[:, :3], p.start, p.kv_len, p.table, max_kv=5000, workspace=p.workspace(4))
    with pytest.raises(RuntimeError, match="device"):
        p.cache.attention(q.cpu(), q, p.start, p.kv_len, p.table, max_kv=5000, workspace=p.workspace(4))
    torch.cuda.synchronize()
