"""Cases of the paged 4-bit key/value cache operators: the step planner (block
tables and slot maps from request lengths), the cache append and read-back, and
attention over the cache for single tokens, drafted tokens and prompts.

Cache format.  uint8 [pages, kv heads, page bytes]; one (page, head) block holds
K codes [P, D/2], K scales [P, D/16], V codes [P, D/2], V scales [P, D/16].  A
code is an e2m1 number (channel 2i in the low four bits of byte i), a scale an
e4m3 number for 16 channels of one token, and a value stands for
code * scale * kv_scales[k or v, head].
"""
import math

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the e2m1 codes 0..7
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------

def listed():
    chain = dict(hq=64, hkv=8, d=128)
    return [
        # one decode step of a small server: 64 running requests, one token each
        dict(name="plan decode", op="plan", n=64, q=1, ctx=4000, page=16),
        # a step that admits many ragged prompts beside running requests
        dict(name="plan prompts", op="plan", n=1000, q=127, ctx=2000, page=32),
        # the new tokens of a decode step, and what the cache then stands for
        dict(name="append decode", op="append", t=16, dtype="f16", page=16, **chain),
        # a long prompt written at once
        dict(name="append prompt", op="append", t=8191, dtype="bf16", page=64, **chain),
        # a short prefix read back in 16 bits
        dict(name="gather prefix", op="gather", t=333, dtype="f16", page=32, hq=16, hkv=4, d=64),
        # a long document handed to a 16-bit cache
        dict(name="gather document", op="gather", t=32769, dtype="bf16", page=16, **chain),
        # the first tokens of one chat: latency alone
        dict(name="decode short", op="attention", n=1, q=1, ctx=16, ragged=False, window=0, dtype="f16", page=16, **chain),
        # one request with a long context: work split along the keys
        dict(name="decode long", op="attention", n=1, q=1, ctx=131070, ragged=False, window=0, dtype="bf16", page=64, **chain),
        # a full server: ragged contexts up to the longest position
        dict(name="decode batch", op="attention", n=64, q=1, ctx=8191, ragged=True, window=0, dtype="bf16", page=16, **chain),
        # five drafted tokens a request, checked together, narrow heads
        dict(name="decode drafts", op="attention", n=16, q=5, ctx=4001, ragged=True, window=0, dtype="f16", page=32,
             hq=16, hkv=4, d=64),
        # a whole prompt from an empty cache
        dict(name="prompt", op="attention", n=1, q=8192, ctx=0, ragged=False, window=0, dtype="f16", page=16, **chain),
        # ragged chunks behind ragged contexts, wide heads, a sliding window
        dict(name="chunks window", op="attention", n=6, q=1000, ctx=3001, ragged=True, window=1024, dtype="bf16", page=64,
             hq=16, hkv=4, d=256),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(("plan", "append", "gather", "decode", "decode", "prompt", "prompt"))
    page = rng.choice((16, 32, 64, 128))
    hq, hkv, d = rng.choice(((64, 8, 128), (8, 1, 128), (16, 4, 64), (16, 4, 256), (32, 32, 128), (28, 4, 128), (4, 2, 256)))
    case = dict(page=page)
    if kind == "plan":
        n = _log(rng, 1, 1000)
        return dict(case, op="plan", n=n, q=rng.choice((1, _log(rng, 1, 127))), ctx=_log(rng, 1, 8000))
    case.update(hq=hq, hkv=hkv, d=d, dtype=rng.choice(("f16", "bf16")))
    if kind in ("append", "gather"):
        return dict(case, op=kind, t=_log(rng, 1, 8191))
    case.update(op="attention", ragged=rng.random() < 0.7, window=rng.choice((0, 0, 0, _log(rng, 16, 4096))))
    if kind == "decode":
        n = _log(rng, 1, 64)
        return dict(case, n=n, q=rng.choice((1, 1, _log(rng, 2, 8))), ctx=_log(rng, 1, min(131070, 4194304 // (n * hkv))))
    n = _log(rng, 1, 8)
    q = _log(rng, 9, 4096 // n)
    return dict(case, n=n, q=q, ctx=_log(rng, 1, 8192 - q))


def _lengths(case):
    """(new tokens, context) of each request: plain numbers of the case alone."""
    n, q, ctx = case["n"], case["q"], case["ctx"]
    if case["op"] == "plan":  # half of a prompt step's requests are new, the others continue
        return [(1 + (i * 37) % q if q > 1 else 1, 0 if q > 1 and i % 2 else 1 + (i * 997) % ctx) for i in range(n)]
    if not case["ragged"] or n == 1:
        return [(q, ctx)] * n
    return [(q if q <= 8 else max(1, q - (q * 5 * ((i * 3) % n)) // (7 * n)), ctx - (ctx * 9 * i) // (10 * n)) for i in range(n)]


def work(case):
    if case["op"] == "plan":
        lens, page = _lengths(case), case["page"]
        need = sum(-(-(c + q) // page) - -(-c // page) for q, c in lens)
        return {"bytes": 4 * (4 * len(lens) + 3 + 2 * need) + 16 * sum(q for q, _ in lens), "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    stored = hkv * (d + d // 8)
    if case["op"] in ("append", "gather"):
        both = case["t"] * (2 * 2 * hkv * d + stored + 8)
        return {"bytes": both * (2 if case["op"] == "append" else 1), "flops": 4 * case["t"] * hkv * d}
    tokens = keys = pairs = 0
    w = case["window"]
    for q, c in _lengths(case):
        tokens += q
        first = max(0, c + 1 - w) if w else 0
        keys += c + q - first
        full = q * (q + 1) // 2 + q * c  # keys that the rows see without a window
        if w:  # less what lies before it: row r sees min(c + r + 1, w)
            over = max(0, c + q - w)
            full -= over * (over + 1) // 2 - (max(0, c - w) * (max(0, c - w) + 1) // 2)
        pairs += full
    return {"bytes": 2 * 2 * tokens * hq * d + keys * stored + 4 * (keys // case["page"]), "flops": 4 * d * hq * pairs}


# ---- inputs ----------------------------------------------------------------------

def _quantize(x, g):
    """(codes 0..15, e4m3 scales) of x [..., D] fp32, g broadcastable to [...]."""
    v = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    g = g[..., None]
    s = (v.abs().amax(-1) / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
    unit = (s.float() * g)[..., None]
    y = torch.where(unit == 0, torch.zeros_like(v), v / unit)
    a = y.abs()
    # halfway points go to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    return code.reshape(x.shape), s


def _parts(cache, page, d):
    """Views of a cache [N, H, bytes]: K codes, K scales, V codes, V scales, each [N, H, page, ...]."""
    n, h, _ = cache.shape
    sizes = (page * d // 2, page * d // 16, page * d // 2, page * d // 16)
    return [p.reshape(n, h, page, -1) for p in cache.split(sizes, -1)]


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _scales(case, gen, dev):
    """Calibrated scales of each head: keys after their norm are near 1, values smaller."""
    u = torch.rand(2, case["hkv"], generator=gen, device=dev)
    return (torch.tensor([[0.9], [0.11]], device=dev) * (0.8 + 0.4 * u)).float()


def _filled(case, gen, dev, pages, valid, g):
    """A cache whose valid slots [pages, page] hold quantised keys and values; the others hold what an
    earlier use left there, with scales that are no numbers."""
    page, hkv, d = case["page"], case["hkv"], case["d"]
    cache = torch.empty(pages, hkv, page * (d + d // 8), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 25) // (hkv * page * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        kc, ks, vc, vs = _parts(cache[a:b], page, d)
        for code, scale, which, size in ((kc, ks, 0, 1.0), (vc, vs, 1, 0.2)):
            x = torch.randn(b - a, hkv, page, d, generator=gen, device=dev) * size
            c, s = _quantize(x, g[which, None, :, None])
            s = s.view(torch.uint8)
            s[~valid[a:b, None, :].expand(-1, hkv, -1)] = 0x7F
            start, width = (0 if which == 0 else page * (d // 2 + d // 16)), page * d // 2
            cache[a:b, :, start:start + width] = _pack(c).reshape(b - a, hkv, -1)
            cache[a:b, :, start + width:start + width + page * d // 16] = s.reshape(b - a, hkv, -1)
    return cache


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    page = case["page"]

    def order(n):
        return torch.randperm(n, generator=gen, device=dev)

    if case["op"] == "plan":
        lens = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[order(case["n"])]
        q, c = lens[:, 0].contiguous(), lens[:, 1].contiguous()
        total = sum(x for x, _ in _lengths(case))
        have = -(-c // page)
        width = -(-(case["ctx"] + case["q"]) // page) + 1
        pool = order(case["n"] * width).int()
        at = torch.arange(width, device=dev)[None, :]
        start = torch.cumsum(have, 0) - have
        table = torch.where(at < have[:, None], pool[(start[:, None] + at).clamp(max=pool.numel() - 1)], -1).int()
        free = pool[int(have.sum()):].contiguous()
        i32 = dict(dtype=torch.int32, device=dev)
        return dict(case=case, query_lens=q, context_lens=c, table=table, free_pages=free,
                    free_count=torch.tensor([free.numel()], **i32), query_start=torch.empty(case["n"] + 1, **i32),
                    seq_lens=torch.empty(case["n"], **i32), free_count_out=torch.empty(1, **i32),
                    positions=torch.empty(total, dtype=torch.int64, device=dev),
                    slots=torch.empty(total, dtype=torch.int64, device=dev))
    hq, hkv, d, dtype = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    g = _scales(case, gen, dev)
    if case["op"] in ("append", "gather"):
        t = case["t"]
        pages = -(-t // page) + 3
        # consecutive tokens of a few requests: whole runs of slots, pages in any order
        slots = (order(pages)[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[:t].contiguous()
        out = dict(key=torch.empty(t, hkv, d, dtype=dtype, device=dev), value=torch.empty(t, hkv, d, dtype=dtype, device=dev))
        if case["op"] == "gather":
            valid = torch.zeros(pages * page, dtype=torch.bool, device=dev)
            valid[slots] = True
            return dict(case=case, cache=_filled(case, gen, dev, pages, valid.view(pages, page), g), scales=g, slots=slots, out=out)
        qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device=dev)
        qkv[:, (hq + hkv) * d:] *= 0.2
        qkv = qkv.to(dtype)
        key = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
        value = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
        cache = torch.zeros(pages, hkv, page * (d + d // 8), dtype=torch.uint8, device=dev)
        return dict(case=case, key=key, value=value, cache=cache, scales=g, slots=slots, out=out)
    lens = _lengths(case)
    lens = [lens[i] for i in order(len(lens)).tolist()]
    tokens, longest = sum(q for q, _ in lens), max(q + c for q, c in lens)
    seq = torch.tensor([q + c for q, c in lens], dtype=torch.int32, device=dev)
    have = -(-seq // page)
    width, pages = -(-longest // page), int(have.sum())
    pool = order(pages).int()
    at = torch.arange(width, device=dev)[None, :]
    first = (torch.cumsum(have, 0) - have)[:, None]
    table = torch.where(at < have[:, None], pool[(first + at).clamp(max=pages - 1)], 0).int()
    slot = torch.arange(width * page, device=dev)[None, :].expand(len(lens), -1)
    valid = torch.zeros(pages * page, dtype=torch.bool, device=dev)
    seen = slot < seq[:, None]
    valid[(table.long().repeat_interleave(page, 1) * page + slot % page)[seen]] = True
    cache = _filled(case, gen, dev, pages, valid.view(pages, page), g)
    qkv = (torch.randn(tokens, (hq + 2 * hkv) * d, generator=gen, device=dev) * 1.5).to(dtype)
    start = torch.tensor([sum(q for q, _ in lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    return dict(case=case, query=qkv[:, :hq * d].view(tokens, hq, d), cache=cache, scales=g, table=table, query_start=start,
                seq_lens=seq, out=torch.empty(tokens, hq, d, dtype=dtype, device=dev), scale=d ** -0.5,
                max_query_len=max(q for q, _ in lens), max_seq_len=longest)


# ---- plain forms -----------------------------------------------------------------

def _values(code, scale, g):
    """fp32 values of packed codes [..., D/2] and scale bytes [..., D/16]; g broadcastable to [...]."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=code.device)
    c = grid[torch.stack((code & 15, code >> 4), -1).long()].reshape(*code.shape[:-1], -1, 16)
    s = scale.contiguous().view(torch.float8_e4m3fn).float()
    return ((c * s[..., None]) * g[..., None, None]).reshape(*code.shape[:-1], -1)


def _plain_plan(s):
    page, q, c = s["case"]["page"], s["query_lens"], s["context_lens"]
    have = (c + page - 1) // page
    need = (c + q + page - 1) // page - have
    table = s["table"]
    fits = have + need <= table.shape[1]
    need = torch.where(fits, need, 0)
    cum = torch.cumsum(need, 0, dtype=torch.int32)
    granted = ((need == 0) | (cum <= s["free_count"])) & fits
    at = torch.arange(table.shape[1], device=q.device)[None, :] - have[:, None]
    new = (at >= 0) & (at < need[:, None]) & granted[:, None]
    taken = s["free_count"] - 1 - ((cum - need)[:, None] + at)
    table = torch.where(new, s["free_pages"][taken.clamp(0, s["free_pages"].numel() - 1)], table)
    end = torch.cumsum(q, 0, dtype=torch.int32)
    start = torch.cat((torch.zeros_like(end[:1]), end))
    t = torch.arange(s["positions"].numel(), device=q.device)
    i = torch.searchsorted(end, t.int(), right=True).clamp(max=q.numel() - 1)
    position = c[i] + t - start[i]
    slot = table[i, (position // page).clamp(max=table.shape[1] - 1)].long() * page + position % page
    slot = torch.where(granted[i], slot, -1)
    count = s["free_count"] - torch.where(granted, cum, 0).amax()
    return dict(query_start=start, seq_lens=torch.where(granted, c + q, ~c), free_count=count, positions=position,
                slots=slot, table=table)


def _plain_gather(s, cache):
    case = s["case"]
    page, d = case["page"], case["d"]
    kc, ks, vc, vs = _parts(cache, page, d)
    p, r = s["slots"] // page, s["slots"] % page
    dtype = DTYPES[case["dtype"]]
    return dict(key=_values(kc[p, :, r], ks[p, :, r], s["scales"][0]).to(dtype),
                value=_values(vc[p, :, r], vs[p, :, r], s["scales"][1]).to(dtype))


def _plain_append(s):
    case = s["case"]
    page, d = case["page"], case["d"]
    cache = s["cache"]
    p, r = s["slots"] // page, s["slots"] % page
    kc, ks, vc, vs = _parts(cache, page, d)  # views: the cache is written in place
    for code, scale, x, g in ((kc, ks, s["key"], s["scales"][0]), (vc, vs, s["value"], s["scales"][1])):
        c, sc = _quantize(x.float(), g)
        code[p, :, r] = _pack(c)
        scale[p, :, r] = sc.view(torch.uint8)
    return _plain_gather(s, cache)


def _plain_attention(s):
    case = s["case"]
    page, d, hkv, w = case["page"], case["d"], case["hkv"], case["window"]
    group = case["hq"] // hkv
    q, seq, start = s["query"], s["seq_lens"], s["query_start"]
    n, width = s["table"].shape
    qmax, keys = s["max_query_len"], width * page
    kc, ks, vc, vs = _parts(s["cache"][s["table"].flatten().long()], page, d)
    where = torch.arange(keys, device=q.device)
    seen = where[None, :] < seq[:, None]

    def rows(code, scale, g):  # [n, hkv, keys, d]; what lies past a request's length does not count
        v = _values(code, scale, g[None, :, None]).view(n, width, hkv, page, d).transpose(1, 2).reshape(n, hkv, keys, d)
        return torch.where(seen[:, None, :, None], v, 0.0)

    k, v = rows(kc, ks, s["scales"][0]), rows(vc, vs, s["scales"][1])
    r = torch.arange(qmax, device=q.device)
    lens = start[1:] - start[:-1]
    token = (start[:-1, None] + r).clamp(max=q.shape[0] - 1).long()
    real = r[None, :] < lens[:, None]
    x = q[token].float().view(n, qmax, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * qmax, d)
    at = (seq - lens)[:, None] + r  # position of each row
    ok = (where[None, None, :] <= at[..., None]) & seen[:, None, :] & real[..., None]
    if w:
        ok &= where[None, None, :] > at[..., None] - w
    score = torch.matmul(x, k.transpose(2, 3)).mul_(s["scale"]).view(n, hkv, group, qmax, keys)
    score.masked_fill_(~ok[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(n, hkv, group * qmax, keys), v).view(n, hkv, group, qmax, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n, qmax, hkv * group, d)
    return o[real].to(q.dtype)


# ---- one pass --------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention,
                "gather": lambda s: _plain_gather(s, s["cache"])}[case["op"]](s)
    import esimd_learning_b200 as ops
    page = case["page"]
    if case["op"] == "plan":
        ops.esimd_kv_plan(s["query_lens"], s["context_lens"], s["table"], s["free_pages"], s["free_count"], page,
                          s["query_start"], s["seq_lens"], s["free_count_out"], s["positions"], s["slots"])
        return dict(query_start=s["query_start"], seq_lens=s["seq_lens"], free_count=s["free_count_out"],
                    positions=s["positions"], slots=s["slots"], table=s["table"])
    if case["op"] == "attention":
        return ops.esimd_kv4_attention(s["query"], s["cache"], s["scales"], s["table"], s["query_start"], s["seq_lens"],
                                       s["out"], page, s["scale"], s["max_query_len"], s["max_seq_len"], case["window"])
    if case["op"] == "append":
        ops.esimd_kv4_append(s["key"], s["value"], s["scales"], s["slots"], s["cache"], page)
    out = s["out"]  # the cache holds 4 bits: what it stands for is read back
    ops.esimd_kv4_gather(s["cache"], s["scales"], s["slots"], out["key"], out["value"], page)
    return out


# ---- in 64 bits ------------------------------------------------------------------

def _decoded(cache, slots, first, page, d, g):
    """float64 [tokens, heads, d] of the K (first = 0) or V part, slot by slot."""
    n, h, width = cache.shape
    code0 = first * page * (d // 2 + d // 16)
    scale0 = code0 + page * d // 2
    row = slots % page
    base = ((slots // page) * h)[:, None] + torch.arange(h, device=slots.device)
    ch = torch.arange(d, device=slots.device)
    flat = cache.reshape(-1)
    byte = flat[(base * width + code0)[..., None] + (row * (d // 2))[:, None, None] + ch // 2].long()
    nib = torch.where(ch % 2 == 0, byte % 16, byte // 16)
    e, m = (nib // 2) % 4, (nib % 2).double()
    mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.pow(2.0, (e - 1).double()))
    sb = flat[(base * width + scale0)[..., None] + (row * (d // 16))[:, None, None] + ch // 16].long()
    se, sm = (sb // 8) % 16, (sb % 8).double()
    scale = torch.where(se == 0, sm / 512, (1 + sm / 8) * torch.pow(2.0, (se - 7).double()))
    return mag * (1 - 2.0 * (nib // 8)) * scale * g.double()[:, None]


def _stored(x, g):
    """What 4 bits keep of x [tokens, heads, d] float64: the nearest number of each grid, ties to the even one."""
    t, h, d = x.shape
    v = x.reshape(t, h, d // 16, 16)
    unit = g.double()[None, :, None]
    a = v.abs().amax(-1) / (6 * unit)
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6))).clamp(max=8.0)
    s = (torch.round(a / torch.pow(2.0, e - 3)) * torch.pow(2.0, e - 3)).clamp(max=448.0)
    y = (v / (s * unit).clamp(min=1e-300)[..., None]).abs().clamp(max=6.0)
    ye = torch.floor(torch.log2(y.clamp(min=1.0)))
    mag = torch.round(y / torch.pow(2.0, ye - 1)) * torch.pow(2.0, ye - 1)
    return (mag.clamp(max=6.0) * v.sign() * (s * unit)[..., None]).reshape(t, h, d)


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers: nothing is rounded
    s = prepare(case, seed)
    page, d, g = case["page"], case["d"], s["scales"]
    if case["op"] == "append":
        return dict(key=_stored(s["key"].double(), g[0]), value=_stored(s["value"].double(), g[1]))
    if case["op"] == "gather":
        return dict(key=_decoded(s["cache"], s["slots"], 0, page, d, g[0]),
                    value=_decoded(s["cache"], s["slots"], 1, page, d, g[1]))
    group, w = case["hq"] // case["hkv"], case["window"]
    starts, seqs = s["query_start"].tolist(), s["seq_lens"].tolist()
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    for i, length in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        if a == b or length <= 0:
            continue
        key = torch.arange(length, device=out.device)
        slots = s["table"][i].long()[key // page] * page + key % page
        k, v = _decoded(s["cache"], slots, 0, page, d, g[0]), _decoded(s["cache"], slots, 1, page, d, g[1])
        at = length - (b - a) + torch.arange(b - a, device=out.device)
        hidden = key[None, :] > at[:, None]
        if w:
            hidden |= key[None, :] <= at[:, None] - w
        for h in range(case["hq"]):
            z = s["query"][a:b, h].double() @ k[:, h // group].T * s["scale"]
            z.masked_fill_(hidden, -math.inf)
            out[a:b, h] = torch.softmax(z, -1) @ v[:, h // group]
    return out
