"""What is measured of the operators for many-stream decoding: the paged 4-bit KV
cache (store), attention over it (single tokens, prompts, sliding window with
sinks) and the per-row draw of next tokens.

`own` false: the operators in elementary torch operations; `own` true: the calls
of this repository's package. Both work on what `prepare` returns.
"""
import random

import torch

own = False

BLOCK = 32          # elements per 4-bit block
D_MAX = 8160.0      # largest scale: 8 * 8160 is still an fp16 number


# ------------------------------------------------------------------ cases ----

def listed():
    """Head layouts and vocabularies are those of the repository's model
    configurations (16/8 heads of 128, 14/2 and 9/3 of 64, 12/12 of 64)."""
    return [
        # one new token of one short conversation: latency alone
        _att("attend_one_short", "f32", 1, 129, 129, 1, 1, 16, 8, 128, 16),
        # a batch of 64 streams, one token each, the repository's streams workload
        _att("attend_streams", "f32", 64, 200, 1600, 1, 1, 16, 8, 128, 32),
        # a full batch of many short and middling streams, half precision, 7 query heads per kv head
        _att("attend_streams_half", "f16", 512, 1, 2100, 1, 1, 14, 2, 64, 64),
        # two long documents, one token each, up to the longest context configured
        _att("attend_long", "f32", 2, 37001, 40960, 1, 1, 16, 8, 128, 64),
        # long conversations that see a window and the first tokens
        _att("attend_window", "f32", 48, 5000, 8192, 1, 1, 9, 3, 64, 16, window=1000, sinks=4),
        # ragged prompts, some of them continuing a cached prefix
        _att("prompt_ragged", "f32", 6, 40, 1200, 1, 512, 16, 8, 128, 16),
        # two long prompts
        _att("prompt_long", "f16", 2, 3900, 4096, 4096, 4096, 16, 8, 128, 64),
        # the keys and values of one step of eight streams
        _store("store_step", "f32", 8, 1, 700, 1, 1, 8, 128, 16),
        # the keys and values of a large prompt batch
        _store("store_prompt", "f16", 5, 1500, 4096, 4096, 4096, 8, 128, 64),
        # one draw of a small vocabulary
        _sample("sample_one", "f32", 1, 32000, "top_k"),
        # a step of 64 streams with everyday settings
        _sample("sample_streams", "f32", 64, 151936, "mixed"),
        # a full batch without truncation
        _sample("sample_full", "f32", 512, 151936, "full"),
    ]


def _att(name, dtype, seqs, kv_min, kv_max, q_min, q_max, heads, kv_heads, head_dim, page, window=0, sinks=0, lens=1):
    return {"name": name, "op": "attention", "dtype": dtype, "seqs": seqs, "kv_min": kv_min, "kv_max": kv_max,
            "q_min": q_min, "q_max": q_max, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "window": window, "sinks": sinks, "lens": lens}


def _store(name, dtype, seqs, kv_min, kv_max, q_min, q_max, kv_heads, head_dim, page, lens=1):
    return {"name": name, "op": "store", "dtype": dtype, "seqs": seqs, "kv_min": kv_min, "kv_max": kv_max,
            "q_min": q_min, "q_max": q_max, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "lens": lens}


def _sample(name, dtype, rows, vocab, mode, lens=1):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "mode": mode, "lens": lens}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


_HEADS = [(16, 8, 128), (14, 2, 64), (9, 3, 64), (12, 12, 64), (8, 1, 32), (3, 1, 32), (4, 2, 64)]


def draw(rng):
    op = rng.choice(["attention", "attention", "prompt", "prompt", "store", "sample", "sample"])
    dtype = rng.choice(["f32", "f16"])
    heads, kv_heads, head_dim = rng.choice(_HEADS)
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1 << 30)
    window, sinks = (0, 0) if rng.random() < 0.5 else (_log_int(rng, 1, 4000), rng.choice([0, 1, 4, 19]))
    if op == "attention":      # one token (sometimes a few) per sequence
        seqs = _log_int(rng, 1, 512)
        kv_max = _log_int(rng, 1, max(2, min(40960, 60000 // seqs)))
        kv_min = _log_int(rng, 1, kv_max)
        q_max = min(rng.choice([1, 1, 1, 2, 5]), kv_max)
        c = _att("", dtype, seqs, kv_min, kv_max, 1, q_max, heads, kv_heads, head_dim, page, window, sinks, lens)
    elif op == "prompt":
        seqs = _log_int(rng, 1, 12)
        kv_max = _log_int(rng, 20, 6000 // seqs + 20)
        kv_min = _log_int(rng, 1, kv_max)
        q_max = _log_int(rng, 10, kv_max)
        c = _att("", dtype, seqs, kv_min, kv_max, rng.choice([1, q_max]), q_max, heads, kv_heads, head_dim, page,
                 window, sinks, lens)
    elif op == "store":
        seqs = _log_int(rng, 1, 64)
        kv_max = _log_int(rng, 1, 16000 // seqs)
        q_max = rng.choice([1, _log_int(rng, 1, kv_max), kv_max])
        c = _store("", dtype, seqs, _log_int(rng, 1, kv_max), kv_max, 1, q_max, kv_heads, head_dim, page, lens)
    else:
        vocab = rng.choice([_log_int(rng, 2, 200000), 32000, 49152, 151936])
        rows = _log_int(rng, 1, max(1, min(512, 40000000 // vocab)))
        c = _sample("", dtype, rows, vocab, rng.choice(["top_k", "mixed", "full", "top_p", "min_p"]), lens)
    del c["name"]
    return c


def _lengths(case):
    """(kv lengths, query lengths) of the case's sequences."""
    r = random.Random(case["lens"])
    kv = [r.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    kv[0] = case["kv_max"]
    q = [min(r.randint(case["q_min"], case["q_max"]), n) for n in kv]
    q[0] = min(case["q_max"], kv[0])
    return kv, q


def _seen(pos, window, sinks):
    """how many positions the row at `pos` sees"""
    n = pos + 1
    return n if window == 0 or n <= window else window + min(sinks, n - window)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * es + case["rows"] * 24, "flops": 4 * n}
    kv, ql = _lengths(case)
    hd, kvh = case["head_dim"], case["kv_heads"]
    pos_bytes = 2 * kvh * hd * 18 // BLOCK       # a position's keys and values in 4 bits
    if case["op"] == "store":
        return {"bytes": sum(ql) * (2 * kvh * hd * es + pos_bytes), "flops": sum(ql) * 2 * kvh * hd * 4}
    read = pairs = 0
    for n, q in zip(kv, ql):
        w, s = case["window"], case["sinks"]
        pairs += sum(_seen(p, w, s) for p in range(n - q, n))
        read += n if w == 0 else min(n, min(s, n) + w + q - 1)
    return {"bytes": read * pos_bytes + 2 * sum(ql) * case["heads"] * hd * es,
            "flops": 4 * hd * case["heads"] * pairs}


# ----------------------------------------------------------------- inputs ----

def _dt(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + case["lens"] % 1000003)
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    kv, ql = _lengths(case)
    kvh, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    r = random.Random(seed)
    need = [-(-n // page) for n in kv]
    pages = list(range(sum(need) + 3))
    r.shuffle(pages)
    table, at = [], 0
    for n in need:
        table.append(pages[at:at + n] + [-1] * (max(need) - n))
        at += n
    start = [0]
    for n in ql:
        start.append(start[-1] + n)
    # keys with a few strong channels, as rotary keys have
    chan = torch.rand(kvh, hd, generator=g, device="cuda") + 0.3
    chan[:, :: max(1, hd // 4)] *= 3.0

    def rows(n, scale):
        return torch.randn(n, kvh, hd, generator=g, device="cuda") * scale
    s = {"case": case, "kv": kv, "ql": ql, "page": page, "table": _i32(table), "start": _i32(start),
         "kv_len": _i32(kv), "n_pages": len(pages)}
    if own:
        import emberllm_b200
        size = emberllm_b200.Kv4Cache.nbytes(len(pages), page, kvh, hd)
        s["cache"] = emberllm_b200.Kv4Cache(torch.zeros(size, dtype=torch.uint8, device="cuda"), len(pages), page, kvh,
                                            hd)
    if case["op"] == "store":
        s["k"] = rows(sum(ql), chan).to(_dt(case))
        s["v"] = rows(sum(ql), 1.0).to(_dt(case))
        if own:
            s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return s
    s["q"] = (torch.randn(sum(ql), case["heads"], hd, generator=g, device="cuda") * 1.2).to(_dt(case))
    total = sum(kv)
    k_code, k_d = _quantize(rows(total, chan))
    v_code, v_d = _quantize(rows(total, 1.0))
    if own:
        # the cache as a program has it: filled by the store of earlier steps
        full = [0]
        for n in kv:
            full.append(full[-1] + n)
        s["cache"].store(_values(k_code, k_d), _values(v_code, v_d), _i32(full), s["kv_len"], s["table"], max(kv))
        s["out"] = torch.empty_like(s["q"])
        size = s["cache"].attention_workspace(case["heads"], len(kv), max(ql), max(kv))
        s["work"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
        return s
    # the plain form's pages: [page, offset, head, ...], two codes to a byte
    slot = torch.cat([_slots(s, i, 0, n) for i, n in enumerate(kv)])
    for name, code, d in (("k", k_code, k_d), ("v", v_code, v_d)):
        packed = torch.zeros(len(pages) * page, kvh, hd // 2, dtype=torch.uint8, device="cuda")
        scale = torch.zeros(len(pages) * page, kvh, hd // BLOCK, dtype=torch.float16, device="cuda")
        packed[slot] = (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)
        scale[slot] = d
        s[name + "_packed"], s[name + "_scale"] = packed, scale
    return s


def _prepare_sample(case, g):
    rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
    # a peaked head over a broad tail, as next-token logits have
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.3
    x += 6.0 * torch.rand(rows, vocab, generator=g, device="cuda") ** 12
    u = torch.rand(rows, generator=g, device="cuda")
    pick = torch.rand(rows, 4, generator=g, device="cuda")
    temperature = 0.5 + pick[:, 0]
    top_k = torch.zeros(rows, dtype=torch.int32, device="cuda")
    top_p = torch.ones(rows, device="cuda")
    min_p = torch.zeros(rows, device="cuda")
    if mode in ("top_k", "mixed"):
        top_k = (1 + pick[:, 1] * 99).to(torch.int32)
    if mode in ("top_p", "mixed"):
        top_p = 0.6 + 0.39 * pick[:, 2]
    if mode == "min_p":
        min_p = 0.001 + 0.2 * pick[:, 3]
    if mode == "mixed":       # every fourth row: top-p alone, min-p alone, greedy, all of them
        i = torch.arange(rows, device="cuda") % 4
        top_k = torch.where(i < 3, torch.zeros_like(top_k), top_k)
        top_p = torch.where(i == 1, torch.ones_like(top_p), top_p)
        min_p = torch.where((i == 1) | (i == 3), 0.001 + 0.1 * pick[:, 3], min_p)
        temperature = torch.where(i == 2, torch.zeros_like(temperature), temperature)
    s = {"case": case, "logits": x.to(_dt(case)), "u": u, "temperature": temperature, "top_k": top_k, "top_p": top_p,
         "min_p": min_p}
    if own:
        s["out"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------- runs ----

def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "sample":
        return _plain_sample(state)
    if case["op"] == "store":
        return _values(*_quantize(state["k"])).to(_dt(case)), _values(*_quantize(state["v"])).to(_dt(case))
    return _plain_attention(state, case)


def _own(s, case):
    if case["op"] == "sample":
        import emberllm_b200
        emberllm_b200.sample_rows(s["logits"], s["out"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                  top_p=s["top_p"], min_p=s["min_p"])
        return s["out"]
    if case["op"] == "store":
        # the cache's own values are read back: what later steps see
        s["cache"].store(s["k"], s["v"], s["start"], s["kv_len"], s["table"], case["q_max"])
        s["cache"].read(s["k_back"], s["v_back"], s["start"], s["kv_len"], s["table"], case["q_max"])
        return s["k_back"], s["v_back"]
    s["cache"].attention(s["q"], s["out"], s["start"], s["kv_len"], s["table"], max_q=case["q_max"],
                         max_kv=case["kv_max"], window=case["window"], sinks=case["sinks"], workspace=s["work"])
    return s["out"]


def _quantize(x):
    """codes and scales of rows of 32-element blocks; 64 bits, since values fall next to borders"""
    x = torch.nan_to_num(x.float(), nan=0.0).double()
    b = x.unflatten(-1, (-1, BLOCK))
    first = b.abs().argmax(-1, keepdim=True)
    d = (torch.gather(b, -1, first) / -8.0).clamp(-D_MAX, D_MAX).to(torch.bfloat16).to(torch.float16)
    dd = d.double()
    code = torch.floor(b / torch.where(dd == 0, 1.0, dd) + 8.5).clamp(0, 15)
    code = torch.where(dd == 0, 8.0, code).to(torch.uint8)
    return code.flatten(-2), d.squeeze(-1)


def _values(code, d):
    return ((code.float() - 8.0).unflatten(-1, (-1, BLOCK)) * d.float().unsqueeze(-1)).flatten(-2)


def _slots(s, i, lo, hi):
    p = torch.arange(lo, hi, device="cuda")
    return s["table"][i].long()[p // s["page"]] * s["page"] + p % s["page"]


def _unpack(packed, scale):
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return _values(code, scale)


def _visible(pos, p, window, sinks):
    see = p <= pos
    if window:
        see = see & ((pos - p < window) | (p < sinks))
    return see


def _plain_attention(s, case):
    if case["q_max"] == 1:
        return _plain_single(s, case)
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.empty_like(s["q"])
    at = 0
    for i, (n, m) in enumerate(zip(s["kv"], s["ql"])):
        slot = _slots(s, i, 0, n)
        k = _unpack(s["k_packed"][slot], s["k_scale"][slot])
        v = _unpack(s["v_packed"][slot], s["v_scale"][slot])
        q = s["q"][at:at + m].float().view(m, kvh, heads // kvh, hd)
        see = _visible(torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None],
                       case["window"], case["sinks"])
        for h in range(kvh):
            score = (q[:, h].transpose(0, 1) @ k[:, h].t()) * hd ** -0.5
            score = score.masked_fill(~see, float("-inf"))
            e = torch.exp(score - score.amax(-1, keepdim=True))
            o = (e / e.sum(-1, keepdim=True)) @ v[:, h]
            out.view(-1, kvh, heads // kvh, hd)[at:at + m, h] = o.transpose(0, 1).to(out.dtype)
        at += m
    return out


def _plain_single(s, case):
    """one token per sequence: sequences padded to the longest, a few at a time"""
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    n, page = case["kv_max"], s["page"]
    out = torch.empty_like(s["q"])
    p = torch.arange(n, device="cuda")
    step = max(1, 200_000_000 // (n * kvh * hd))
    for a in range(0, case["seqs"], step):
        t = s["table"][a:a + step].long().clamp(min=0)
        slot = t[:, p // page] * page + p % page
        k = _unpack(s["k_packed"][slot], s["k_scale"][slot]).permute(0, 2, 1, 3)
        v = _unpack(s["v_packed"][slot], s["v_scale"][slot]).permute(0, 2, 1, 3)
        q = s["q"][a:a + step].float().view(-1, kvh, heads // kvh, hd)
        see = _visible((s["kv_len"][a:a + step].long() - 1)[:, None], p[None], case["window"], case["sinks"])
        score = (q @ k.transpose(-1, -2)) * hd ** -0.5
        score = score.masked_fill(~see[:, None, None], float("-inf"))
        e = torch.exp(score - score.amax(-1, keepdim=True))
        out[a:a + step] = ((e / e.sum(-1, keepdim=True)) @ v).reshape(-1, heads, hd).to(out.dtype)
    return out


def _plain_sample(s):
    """one draw per row; sums in 64 bits, since the draw falls next to borders"""
    x = s["logits"].float()
    t = s["temperature"][:, None].double()
    l, index = torch.sort(x, dim=-1, descending=True, stable=True)
    d = (l.double() - l[:, :1].double()) / torch.where(t > 0, t, 1.0)
    w = torch.exp(d)
    run_sum = torch.cumsum(w, -1)
    rank = torch.arange(x.shape[1], device="cuda")[None]
    k, p, m = s["top_k"][:, None], s["top_p"][:, None].double(), s["min_p"][:, None].double()
    keep = (rank < k) | (k <= 0)
    keep &= (w >= m) | (m <= 0) | (m >= 1)
    before = run_sum - w
    keep &= (before < p * run_sum[:, -1:]) | (p <= 0) | (p >= 1)
    last = keep.sum(-1, keepdim=True) - 1
    r = s["u"][:, None].double() * torch.gather(run_sum, -1, last)
    chosen = torch.minimum((run_sum <= r).sum(-1, keepdim=True), last)
    chosen = torch.where(t > 0, chosen, 0)
    return torch.gather(index, -1, chosen)[:, 0].to(torch.int32)


# ------------------------------------------------------------------ exact ----

def exact(case, seed):
    """the definitions in 64 bits; tokens of a draw are whole numbers and have no such value"""
    global own
    if case["op"] == "sample":
        return None
    mode, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mode
    if case["op"] == "store":
        return _exact_blocks(s["k"]), _exact_blocks(s["v"])
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    group = heads // kvh
    if work(case)["flops"] > 4e12:
        return None
    rows = []
    at = 0
    for i, (n, m) in enumerate(zip(s["kv"], s["ql"])):
        where = _slots(s, i, 0, n)
        kv = []
        for name in ("k", "v"):
            byte = s[name + "_packed"][where].to(torch.int64)
            value = torch.empty(n, kvh, hd, dtype=torch.float64, device="cuda")
            value[..., 0::2] = (byte % 16 - 8).double()
            value[..., 1::2] = (byte // 16 - 8).double()
            kv.append(value * s[name + "_scale"][where].double().repeat_interleave(BLOCK, -1))
        col = torch.arange(n, device="cuda")
        row = torch.arange(n - m, n, device="cuda").unsqueeze(1)
        hidden = col > row
        if case["window"] > 0:
            hidden |= (col <= row - case["window"]) & (col >= case["sinks"])
        seq = torch.empty(m, heads, hd, dtype=torch.float64, device="cuda")
        for h in range(heads):
            z = torch.einsum("md,nd->mn", s["q"][at:at + m, h].double(), kv[0][:, h // group]) / hd ** 0.5
            z[hidden] = -torch.inf
            z = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
            seq[:, h] = torch.einsum("mn,nd->md", z, kv[1][:, h // group])
        rows.append(seq)
        at += m
    return torch.cat(rows)


def _exact_blocks(x):
    """each 32-element block: the value of largest magnitude becomes -8 steps, the others the nearest step"""
    a = x.double().reshape(-1, BLOCK)
    hi, lo = a.max(1).values, a.min(1).values
    peak = torch.where(hi > -lo, hi, lo)
    both = hi == -lo
    if both.any():      # the first of the two decides
        sub = a[both]
        peak[both] = torch.gather(sub, 1, (sub.abs() == hi[both, None]).int().argmax(1, keepdim=True))[:, 0]
    step = (-peak / 8).clamp(-D_MAX, D_MAX).to(torch.bfloat16).to(torch.float16).double()[:, None]
    n = torch.where(step == 0, 0.0, torch.floor(a / torch.where(step == 0, 1.0, step) + 0.5).clamp(-8, 7))
    return (n * step).reshape(x.shape)
