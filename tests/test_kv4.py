"""The paged 4-bit key/value cache: page plan, append, read-back and attention
against oracle/kv4.py, at the sizes, masks and layouts where they can go wrong,
and their refusals.

Attention's tolerance, per element: the output's own rounding u |o| (u = 2^-11
for fp16, 2^-8 for bf16, 2^-25 at least: fp16 subnormals), the fp16 rounding of
the probabilities, 2^-11 of the largest value that the row sees (the
probabilities sum to one), and fp32 arithmetic: scores of magnitude S (log2
units) carry an error of some 2^-22 S, which moves a probability by that
relative amount; S stays below 2^8 here, so 2^-13 of the largest value covers
it and the sums.
"""
import ctypes

import pytest
import torch

from esimd_learning_b200 import cabi
from oracle import kv4 as K

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def tolerance(ref, vmax, dtype):
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    return u * ref.abs() + (2.0 ** -11 + 2.0 ** -13) * vmax[..., None] + 2.0 ** -25


def scales_for(hkv, gen):
    return (torch.tensor([[0.9], [0.11]]) * (0.8 + 0.4 * torch.rand(2, hkv, generator=gen))).float()


def page_bytes(page, d):
    return page * (d + d // 8)


# ---- no GPU ----------------------------------------------------------------------

def test_oracle_quantiser_bounds():
    """The kept value is within half a step of the input: at most unit / 2 below 2 units and unit / 4 ... 1
    above, with unit within 1/16 (e4m3) of max / 6 — 0.25 of the group's maximum covers every grid gap."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(50, 3, 64, generator=gen).half()
    g = torch.tensor([1.0, 0.3, 2.0])
    code, scale = K.quantize(x, g)
    nib = torch.stack((code & 15, code >> 4), -1).reshape(50, 3, 64).numpy()
    val = K.E2M1[nib & 7] * (1 - 2.0 * (nib >> 3)) * K.E4M3[scale.numpy()].repeat(16, -1) * g.numpy()[None, :, None]
    top = x.float().reshape(50, 3, 4, 16).abs().amax(-1).repeat_interleave(16, -1)
    assert ((torch.from_numpy(val) - x.double()).abs() <= 0.25 * top).all()


def test_oracle_grids():
    assert torch.tensor(K.E4M3[:127]).float().to(torch.float8_e4m3fn).view(torch.uint8).tolist() == list(range(127))
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    import numpy as np
    assert K.nearest_even(np.array(ties), K.E2M1).tolist() == [0, 2, 2, 4, 4, 6, 6]


def test_oracle_plan_by_hand():
    # page 4; request 0 has 3 of 4 slots filled, 1 is refused for want of pages, 2 needs none
    t, s, seq, left, pos, slots = K.plan([2, 9, 1], [3, 0, 5], [[7, 0, 0], [0, 0, 0], [8, 9, 0]], [1, 2, 3], 3, 4, 13)
    assert t == [[7, 3, 0], [0, 0, 0], [8, 9, 0]] and s == [0, 2, 11, 12] and seq == [5, -1, 6] and left == 2
    assert pos == [3, 4, *range(9), 5, 0] and slots == [31, 12] + [-1] * 9 + [37, -1]


def _cache(**kw):
    c = cabi.Kv4Cache(16, 16, 4, 2 * page_bytes(16, 64), page_bytes(16, 64), 2, 64, 16)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def _attend(cache=None, **kw):
    a = dict(q=16, table=16, start=16, seq=16, out=16, ws=16, wsb=1 << 40, B=1, T=1, hq=4, W=1, ts=1, qts=256, qhs=64,
             ots=256, ohs=64, scale=0.125, mq=1, ms=16, window=0, dt=0)
    a.update(kw)
    return cabi.lib().cek_kv4_attention(
        a["q"], cache or _cache(), a["table"], a["start"], a["seq"], a["out"], a["ws"], a["wsb"], a["B"], a["T"], a["hq"],
        a["W"], a["ts"], a["qts"], a["qhs"], a["ots"], a["ohs"], a["scale"], a["mq"], a["ms"], a["window"], a["dt"], None)


@pytest.mark.parametrize("kw", [dict(q=0), dict(out=0), dict(table=0), dict(start=0), dict(seq=0), dict(B=-1), dict(T=-1),
                                dict(hq=3), dict(hq=0), dict(W=-1), dict(ts=0), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(mq=-1), dict(ms=-1),
                                dict(window=-1), dict(dt=2)])
def test_attention_refuses(kw):
    assert _attend(**kw) == cabi.CEK_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(q=8), dict(out=24), dict(qts=252), dict(qhs=60), dict(ots=260), dict(ohs=68)])
def test_attention_refuses_alignment(kw):
    assert _attend(**kw) == cabi.CEK_ERR_ALIGNMENT


def test_attention_of_nothing_is_ok():
    assert _attend(B=0) == cabi.CEK_OK and _attend(T=0) == cabi.CEK_OK and _attend(mq=0) == cabi.CEK_OK


BAD_CACHES = [dict(head_dim=96), dict(page_size=48), dict(page_size=8), dict(num_pages=0), dict(kv_heads=0),
              dict(data=None), dict(scales=None), dict(head_stride=16), dict(page_stride=page_bytes(16, 64) - 16)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_cache_refusals(kw):
    L = cabi.lib()
    assert _attend(_cache(**kw)) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_append(16, 16, 16, _cache(**kw), 1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_gather(_cache(**kw), 16, 16, 16, 1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_INVALID_ARG


def test_token_op_refusals():
    L = cabi.lib()
    assert L.cek_kv4_append(0, 16, 16, _cache(), 1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_append(16, 16, 0, _cache(), 1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_append(16, 16, 16, _cache(), -1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_append(16, 16, 16, _cache(), 1, 128, 64, 128, 64, 3, None) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_append(16, 16, 16, _cache(data=24), 1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_ALIGNMENT
    assert L.cek_kv4_append(0, 0, 0, _cache(), 0, 128, 64, 128, 64, 0, None) == cabi.CEK_OK
    assert L.cek_kv4_gather(_cache(), 16, 16, 0, 1, 128, 64, 128, 64, 0, None) == cabi.CEK_ERR_INVALID_ARG
    assert L.cek_kv4_page_bytes(16, 128) == 2304 and L.cek_kv4_page_bytes(24, 128) == 0 and L.cek_kv4_page_bytes(16, 80) == 0


def _plan(**kw):
    a = dict(q=16, c=16, table=16, pool=16, count=16, start=16, seq=16, out=16, pos=16, slots=16, B=1, W=1, ts=1, F=1,
             T=1, P=16)
    a.update(kw)
    return cabi.lib().cek_kv_plan(*(a[k] for k in ("q", "c", "table", "pool", "count", "start", "seq", "out", "pos",
                                                   "slots", "B", "W", "ts", "F", "T", "P")), None)


@pytest.mark.parametrize("kw", [dict(q=0), dict(c=0), dict(table=0), dict(pool=0), dict(count=0), dict(start=0),
                                dict(seq=0), dict(out=0), dict(pos=0), dict(slots=0), dict(B=-1), dict(B=4097),
                                dict(W=2), dict(F=-1), dict(T=-1), dict(P=0)])
def test_plan_refuses(kw):
    assert _plan(**kw) == cabi.CEK_ERR_INVALID_ARG


def test_ops_registered_and_fail_on_cpu(ext):
    for name in ("esimd_kv_plan", "esimd_kv4_append", "esimd_kv4_gather", "esimd_kv4_attention"):
        assert hasattr(torch.ops.custom_esimd_kernels_vllm, name) and callable(getattr(ext, name))
    k = torch.zeros(1, 1, 64).half()
    with pytest.raises(NotImplementedError):
        ext.esimd_kv4_append(k, k, torch.ones(2, 1), torch.zeros(1, dtype=torch.int64),
                             torch.zeros(1, 1, page_bytes(16, 64), dtype=torch.uint8), 16)


# ---- page plan -------------------------------------------------------------------

def run_plan(ext, dev, q, c, table, pool, count, page, tokens, alias=False):
    i32 = dict(dtype=torch.int32, device=dev)
    width = len(table[0]) if table else 0
    tq, tc = torch.tensor(q, **i32), torch.tensor(c, **i32)
    tt = torch.tensor(table, **i32).view(len(q), width)
    fp, fc = torch.tensor(pool, **i32), torch.tensor([count], **i32)
    start = torch.full((len(q) + 1,), -7, **i32)
    seq = tc if alias else torch.full_like(tc, -7)
    left = fc if alias else torch.full_like(fc, -7)
    pos = torch.full((tokens,), -7, dtype=torch.int64, device=dev)
    slots = torch.full((tokens,), -7, dtype=torch.int64, device=dev)
    ext.esimd_kv_plan(tq, tc, tt, fp, fc, page, start, seq, left, pos, slots)
    return tt.tolist(), start.tolist(), seq.tolist(), left.item(), pos.tolist(), slots.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("B,qmax,cmax,page", [(1, 1, 0, 16), (1, 1, 15, 16), (1, 40, 16, 16), (5, 1, 100, 32),
                                              (33, 9, 300, 64), (1023, 3, 50, 16), (1025, 7, 200, 128), (4096, 5, 64, 16),
                                              (7, 3000, 10, 16), (9, 9000, 50, 32), (3, 9, 20, 1), (6, 11, 40, 12)])
@pytest.mark.parametrize("room", ["enough", "short", "none"])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(ext, cuda_device, B, qmax, cmax, page, room, alias):
    gen = torch.Generator().manual_seed(B * 31 + qmax)
    q = torch.randint(0, qmax + 1, (B,), generator=gen).tolist()
    c = torch.randint(0, cmax + 1, (B,), generator=gen).tolist()
    for i in range(0, B, 11):
        c[i] = ~c[i] if i else c[i]  # refused before
    width = -(-(cmax + qmax) // page)
    width -= 1 if width > 2 and room == "short" else 0  # some rows are too narrow
    have = [-(-max(x, 0) // page) for x in c]
    pages = torch.randperm(B * (width + 2) + 8, generator=gen).tolist()
    table = [[pages.pop() if j < have[i] else -1 for j in range(width)] for i in range(B)]
    want = sum(-(-(max(a, 0) + b) // page) for a, b in zip(c, q)) - sum(have)
    count = {"enough": len(pages) - 3, "short": want // 2, "none": 0}[room]
    tokens = sum(q) + (5 if B % 2 else 0)  # padded, or exact
    ref = K.plan(q, c, table, pages, count, page, tokens)
    got = run_plan(ext, cuda_device, q, c, table, pages, count, page, tokens, alias)
    assert got == tuple(ref)


@pytest.mark.gpu
def test_plan_of_nothing(ext, cuda_device):
    got = run_plan(ext, cuda_device, [], [], [], [3, 4], 2, 16, 3)
    assert got == ([], [0], [], 2, [0, 0, 0], [-1, -1, -1])


@pytest.mark.gpu
def test_plan_drops_tokens_past_the_outputs(ext, cuda_device):
    got = run_plan(ext, cuda_device, [5, 5], [0, 0], [[-1], [-1]], [3, 4], 2, 16, 7)
    assert got == ([[4], [3]], [0, 5, 10], [5, 5], 0, [0, 1, 2, 3, 4, 0, 1], [64, 65, 66, 67, 68, 48, 49])


@pytest.mark.gpu
def test_plan_strided_table_and_wrong_arguments(ext, cuda_device):
    i32 = dict(dtype=torch.int32, device=cuda_device)
    big = torch.full((3, 8), -1, **i32)
    args = lambda table: (torch.ones(3, **i32), torch.zeros(3, **i32), table, torch.arange(9, **i32), torch.tensor([9], **i32),  # noqa: E731
                          16, torch.zeros(4, **i32), torch.zeros(3, **i32), torch.zeros(1, **i32),
                          torch.zeros(3, dtype=torch.int64, device=cuda_device), torch.zeros(3, dtype=torch.int64, device=cuda_device))
    ext.esimd_kv_plan(*args(big[:, 2:5]))
    assert big.tolist() == [[-1, -1, v, -1, -1, -1, -1, -1] for v in (8, 7, 6)]
    with pytest.raises(RuntimeError):
        ext.esimd_kv_plan(*args(big.t()[:3]))
    with pytest.raises(RuntimeError):
        ext.esimd_kv_plan(*args(big[:2]))
    with pytest.raises(RuntimeError):
        ext.esimd_kv_plan(*args(big.long()))


# ---- append and gather -----------------------------------------------------------

def special(x):
    """Values where a quantiser goes wrong, in the first tokens: zeros of both signs, infinities, NaN, tiny, huge, ties."""
    t = x.shape[0]
    f = torch.finfo(x.dtype)
    if t > 1:
        x[1, 0, :16] = 0.0
        x[1, 0, 16:32] = -0.0
        x[1, 0, 32:48] = f.tiny / 8
    if t > 2:
        x[2, 0, 3] = float("inf")
        x[2, 0, 20] = float("-inf")
        x[2, -1, 5] = float("nan")
    if t > 3:
        x[3, 0] = torch.linspace(-6, 6, x.shape[2]).to(x.dtype)
        x[3, -1, :16] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0])
        x[3, -1, 16:32] = f.max
    return x


def cache_case(T, hkv, d, page, dtype, seed, hq=2, g=None):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=gen)
    qkv[:, (hq + hkv) * d:] *= 0.1
    qkv = qkv.to(dtype)
    k = special(qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d))
    v = special(qkv[:, (hq + hkv) * d:].view(T, hkv, d))
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=gen)[:T]
    scales = scales_for(hkv, gen) if g is None else torch.full((2, hkv), g)
    cache = torch.randint(0, 256, (pages, hkv, page_bytes(page, d)), generator=gen, dtype=torch.uint8)
    return qkv, k, v, slots, scales, cache


APPEND = [(1, 1, 64, 16, "f16"), (5, 2, 64, 32, "bf16"), (17, 8, 128, 16, "bf16"), (33, 4, 128, 64, "f16"),
          (130, 1, 256, 128, "f16"), (9, 3, 256, 16, "bf16")]


@pytest.mark.gpu
@pytest.mark.parametrize("T,hkv,d,page,dt", APPEND)
@pytest.mark.parametrize("g", [None, 1.0, 2.0 ** -30, 3e4])
def test_append_bits(ext, cuda_device, T, hkv, d, page, dt, g):
    qkv, k, v, slots, scales, cache = cache_case(T, hkv, d, page, DT[dt], 1, g=g)
    if T > 4:
        slots[4], slots[0] = -1, cache.shape[0] * page  # skipped
    ref = K.append(cache, page, k, v, scales, slots)
    dq = qkv.to(cuda_device)
    hq = 2
    dc = cache.to(cuda_device)
    ret = ext.esimd_kv4_append(dq[:, hq * d:(hq + hkv) * d].view(T, hkv, d), dq[:, (hq + hkv) * d:].view(T, hkv, d),
                               scales.to(cuda_device), slots.to(cuda_device), dc, page)
    assert ret.data_ptr() == dc.data_ptr()
    assert torch.equal(dc.cpu(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("T,hkv,d,page,dt", APPEND)
def test_gather(ext, cuda_device, T, hkv, d, page, dt):
    _, _, _, slots, scales, cache = cache_case(T, hkv, d, page, DT[dt], 2)
    if T > 4:
        slots[4], slots[0], slots[3] = -1, cache.shape[0] * page, slots[2]  # nothing, nothing, twice
    ok = (slots >= 0) & (slots < cache.shape[0] * page)
    out = [torch.full((T, hkv, d), 7.0, dtype=DT[dt], device=cuda_device) for _ in range(2)]
    ext.esimd_kv4_gather(cache.to(cuda_device), scales.to(cuda_device), slots.to(cuda_device), *out, page)
    for part in (0, 1):
        # code * scale is exact in fp32: one fp32 rounding, one to the output type
        ref = torch.from_numpy(K.decode(cache, page, d, torch.where(ok, slots, 0).numpy(), part, scales))
        ref = torch.where(ok[:, None, None], ref, 0.0).float().to(DT[dt])
        got = out[part].cpu()
        assert torch.equal(torch.nan_to_num(got, 1234.0), torch.nan_to_num(ref, 1234.0))


@pytest.mark.gpu
def test_append_gather_strides_and_alignment(ext, cuda_device):
    """Views off a 16-byte boundary, heads before tokens, a cache that is a slice of all layers' pages."""
    T, hkv, d, page = 21, 3, 64, 16
    _, k, v, slots, scales, cache = cache_case(T, hkv, d, page, torch.float16, 3)
    ref = K.append(cache, page, k, v, scales, slots)
    dev = cuda_device
    layers = torch.zeros(cache.shape[0], 2, hkv, page_bytes(page, d), dtype=torch.uint8, device=dev)
    dc = layers[:, 1]
    dc.copy_(cache)
    flat = torch.zeros(hkv, T, d + 3, dtype=torch.float16, device=dev)
    kk = flat[:, :, 1:1 + d].transpose(0, 1)
    kk.copy_(k)
    vv = v.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    ext.esimd_kv4_append(kk, vv, scales.to(dev), slots.to(dev), dc, page)
    assert torch.equal(dc.cpu(), ref) and not layers[:, 0].any()
    ko = torch.zeros(hkv, T, d + 3, dtype=torch.float16, device=dev)[:, :, 1:1 + d].transpose(0, 1)
    vo = torch.zeros(T, hkv, d, dtype=torch.float16, device=dev)
    ext.esimd_kv4_gather(dc, scales.to(dev), slots.to(dev), ko, vo, page)
    for part, got in ((0, ko), (1, vo)):
        want = torch.from_numpy(K.decode(ref, page, d, slots.numpy(), part, scales)).float().half()
        assert torch.equal(torch.nan_to_num(got.cpu(), 1234.0), torch.nan_to_num(want, 1234.0))


@pytest.mark.gpu
def test_token_op_wrong_tensors(ext, cuda_device):
    dev = cuda_device
    k = torch.zeros(2, 1, 64, dtype=torch.float16, device=dev)
    s, slots = torch.ones(2, 1, device=dev), torch.arange(2, device=dev)
    c = torch.zeros(1, 1, page_bytes(16, 64), dtype=torch.uint8, device=dev)
    ext.esimd_kv4_append(k, k, s, slots, c, 16)
    for bad in [(k.float(), k, s, slots, c, 16), (k, k.bfloat16(), s, slots, c, 16), (k, k[:1], s, slots, c, 16),
                (k, k, s.half(), slots, c, 16), (k, k, s[:1], slots, c, 16), (k, k, s, slots.int(), c, 16),
                (k, k, s, slots[:1], c, 16), (k, k, s, slots, c[..., :-16], 16), (k, k, s, slots, c, 32),
                (k, k, s, slots, c.int(), 16), (k.transpose(0, 2), k, s, slots, c, 16), (k, k, s.cpu(), slots, c, 16)]:
        with pytest.raises(RuntimeError):
            ext.esimd_kv4_append(*bad)


# ---- attention -------------------------------------------------------------------

def attention_case(lens, hq, hkv, d, page, dtype, seed=0, size=1.5, stale=0xFF):
    """lens: (new tokens, total tokens) of each request.  Slots that hold no token are `stale` bytes (NaN scales)."""
    gen = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-max(n, 0) // page) for _, n in lens))
    used = [-(-max(n, 0) // page) for _, n in lens]
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.tensor([[order.pop() if j < u else -1 for j in range(width)] for u in used], dtype=torch.int32)
    scales = scales_for(hkv, gen)
    cache = torch.full((pages, hkv, page_bytes(page, d)), stale, dtype=torch.uint8)
    slots = torch.tensor([table[i, j // page].item() * page + j % page for i, (_, n) in enumerate(lens) for j in range(max(n, 0))],
                         dtype=torch.int64)
    k = torch.randn(len(slots), hkv, d, generator=gen).to(dtype)
    v = (torch.randn(len(slots), hkv, d, generator=gen) * 0.2).to(dtype)
    off = K.offsets(page, d)
    for part, x in ((0, k), (1, v)):
        code, scale = K.quantize(x, scales[part])
        p, r = slots // page, slots % page
        n = cache.shape[0]
        cache[:, :, off[2 * part]:off[2 * part] + page * d // 2].view(n, hkv, page, d // 2)[p, :, r] = code
        cache[:, :, off[2 * part + 1]:off[2 * part + 1] + page * d // 16].view(n, hkv, page, d // 16)[p, :, r] = scale
    T = sum(q for q, _ in lens)
    q = (torch.randn(T, hq, d, generator=gen) * size).to(dtype)
    start = torch.tensor([sum(x for x, _ in lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    seq = torch.tensor([n for _, n in lens], dtype=torch.int32)
    return dict(q=q, cache=cache, scales=scales, table=table, start=start, seq=seq, page=page, scale=d ** -0.5,
                max_q=max(q for q, _ in lens), max_seq=max(n for _, n in lens))


def run_attention(ext, dev, c, window=0, max_q=None, max_seq=None, out=None):
    out = torch.full_like(c["q"], 77.0, device=dev) if out is None else out
    ext.esimd_kv4_attention(c["q"].to(dev), c["cache"].to(dev), c["scales"].to(dev), c["table"].to(dev), c["start"].to(dev),
                            c["seq"].to(dev), out, c["page"], c["scale"], c["max_q"] if max_q is None else max_q,
                            max(c["max_seq"], 0) if max_seq is None else max_seq, window)
    return out


def check_attention(ext, dev, c, window=0, **kw):
    got = run_attention(ext, dev, c, window, **kw).cpu()
    ref, vmax = K.attention(c["q"], c["cache"], c["page"], c["scales"], c["table"], c["start"], c["seq"], c["scale"], window)
    assert torch.isfinite(got).all()
    err = (got.double() - ref).abs()
    bad = err > tolerance(ref, vmax, got.dtype)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (err / tolerance(ref, vmax, got.dtype)).max().item())
    return got


HEADS = [(1, 1, 64), (16, 4, 64), (64, 8, 128), (8, 1, 128), (4, 2, 256), (3, 3, 128), (28, 4, 128), (20, 1, 64), (40, 2, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_single_tokens(ext, cuda_device, hq, hkv, d, page, dt):
    """One token a request: a single key, either side of a page and of 64 keys, no keys, a refused request."""
    lens = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 0), (1, 63), (1, 64), (1, 65), (1, -6), (1, 129), (1, 300)]
    got = check_attention(ext, cuda_device, attention_case(lens, hq, hkv, d, page, DT[dt]))
    assert not got[4].any() and not got[8].any()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,page", [(64, 8, 128, 16), (16, 4, 64, 32), (4, 2, 256, 64), (5, 5, 128, 128), (12, 1, 64, 16)])
@pytest.mark.parametrize("window", [0, 1, 7, 100])
def test_attention_drafts(ext, cuda_device, hq, hkv, d, page, window):
    """A few tokens a request (some none), rows that see nothing, windows."""
    lens = [(3, 3), (5, 70), (0, 9), (2, 0), (8, 40), (1, 200), (4, 2), (7, 129)]
    got = check_attention(ext, cuda_device, attention_case(lens, hq, hkv, d, page, torch.float16), window)
    assert not got[8:10].any() and not got[19:21].any()  # an empty request; the two rows before position 0


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 1, 128, 16), (4, 4, 64, 64), (4, 2, 256, 32), (7, 1, 128, 128), (2, 1, 64, 16)])
@pytest.mark.parametrize("window", [0, 1, 50, 200])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_prompts(ext, cuda_device, hq, hkv, d, page, window, dt):
    """Ragged prompts and chunks: odd lengths, behind a context, none, tiles that end anywhere."""
    lens = [(130, 130), (33, 97), (1, 50), (0, 5), (257, 300), (64, 64), (17, 0), (20, 500), (9, 6)]
    check_attention(ext, cuda_device, attention_case(lens, hq, hkv, d, page, DT[dt]), window)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1000, 4097, 20001])
@pytest.mark.parametrize("hq,hkv,d,q", [(8, 1, 128, 1), (4, 2, 256, 3), (4, 1, 64, 40)])
def test_attention_long(ext, cuda_device, n, hq, hkv, d, q):
    """A long axis beside a short one: work split along the keys and joined."""
    c = attention_case([(q, n), (q, n // 7)], hq, hkv, d, 64, torch.bfloat16)
    got = check_attention(ext, cuda_device, c)
    assert torch.equal(got, run_attention(ext, cuda_device, c).cpu())  # the same bits every time
    check_attention(ext, cuda_device, c, max_seq=n + 10000)  # a loose bound


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 4, 150])
def test_attention_peaked_and_flat(ext, cuda_device, q):
    """Scores far apart (one key takes all) and all equal (queries of zeros)."""
    c = attention_case([(q, 700), (q, 160)], 8, 2, 128, 16, torch.float16, size=6.0)
    check_attention(ext, cuda_device, c)
    c["q"].zero_()
    check_attention(ext, cuda_device, c)


@pytest.mark.gpu
def test_attention_query_ranges(ext, cuda_device):
    """bf16 queries beyond fp16's range on both sides."""
    c = attention_case([(1, 100), (3, 90), (140, 150)], 8, 2, 64, 16, torch.bfloat16)
    c["q"][0] *= 2.0 ** 100
    c["q"][1:3] *= 2.0 ** -60
    c["q"][2, :, 5] = 1.0
    c["scale"] = 2.0 ** -100
    c["q"][4:] *= 2.0 ** 97
    check_attention(ext, cuda_device, c)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 3, 150])
def test_attention_strides(ext, cuda_device, q):
    """Queries and outputs inside wider rows, a cache that is one layer of many, a wide table."""
    c = attention_case([(q, 200), (q, 151)], 8, 2, 128, 32, torch.float16)
    ref = run_attention(ext, cuda_device, c).cpu()
    T = c["q"].shape[0]
    wide = torch.zeros(T, 12, 136, dtype=torch.float16, device=cuda_device)
    qv = wide[:, 2:10, 8:]
    qv.copy_(c["q"])
    out = torch.full((8, T, 128), 5.0, dtype=torch.float16, device=cuda_device).transpose(0, 1)
    layers = torch.full((c["cache"].shape[0], 3, *c["cache"].shape[1:]), 0xFF, dtype=torch.uint8, device=cuda_device)
    layers[:, 1] = c["cache"].to(cuda_device)
    table = torch.full((2, 50), -1, dtype=torch.int32, device=cuda_device)
    table[:, 3:3 + c["table"].shape[1]] = c["table"].to(cuda_device)
    c2 = dict(c, q=qv, cache=layers[:, 1], table=table[:, 3:])
    got = run_attention(ext, cuda_device, c2, out=out).cpu()
    assert torch.equal(got, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 2, 130])
def test_attention_offsets_past_32_bits(ext, cuda_device, q):
    c = attention_case([(q, 140)], 2, 1, 64, 16, torch.float16)
    n, hkv, block = c["cache"].shape
    stride = (3 << 30) // 16 * 16
    big = torch.empty(stride * (n - 1) + block, dtype=torch.uint8, device=cuda_device)
    view = big.as_strided((n, hkv, block), (stride, block, 1))
    view.copy_(c["cache"])
    assert torch.equal(run_attention(ext, cuda_device, dict(c, cache=view)).cpu(), run_attention(ext, cuda_device, c).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("q", [2, 6, 140])
def test_attention_nan_behind_a_row_stays_there(ext, cuda_device, q):
    """The last token's key and value are NaN: only the last row sees them; the value's NaN in one group of 16."""
    n, d, page = 150, 64, 16
    c = attention_case([(q, n), (q, n - 3)], 4, 1, d, page, torch.float16)
    ref = run_attention(ext, cuda_device, c).cpu()
    off = K.offsets(page, d)
    slot = c["table"][0, (n - 1) // page].item(), (n - 1) % page
    c["cache"][slot[0], 0, off[3] + slot[1] * (d // 16) + 2] = 0x7F
    got = run_attention(ext, cuda_device, c).cpu()
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[q - 1, :, 32:48] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], ref[~nan])
    c["cache"][slot[0], 0, off[1] + slot[1] * (d // 16) + 1] = 0xFF
    got = run_attention(ext, cuda_device, c).cpu()
    nan[q - 1] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], ref[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 3, 140])
def test_attention_nan_query_stays_in_its_row(ext, cuda_device, q):
    c = attention_case([(q, 150), (q, 149)], 4, 2, 64, 16, torch.bfloat16)
    ref = run_attention(ext, cuda_device, c).cpu()
    c["q"][0, 1, 3] = float("nan")
    got = run_attention(ext, cuda_device, c).cpu()
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = ref[0, 1]
    assert torch.equal(got, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 2, 150])
def test_attention_bounds_cut(ext, cuda_device, q):
    """Bounds below a request's lengths: the rows past max_query_len are not written, the keys past max_seq_len not read."""
    c = attention_case([(q, 200), (q, 160)], 4, 2, 128, 16, torch.float16)
    full = run_attention(ext, cuda_device, c).cpu()
    if q > 1:
        got = run_attention(ext, cuda_device, c, max_q=q - 1).cpu()
        assert (got[q - 1] == 77).all() and torch.equal(got[:q - 1], full[:q - 1])
    cut = run_attention(ext, cuda_device, c, max_seq=40).cpu()
    # rows at or past position 39 see the keys 0 .. 39 in both requests
    ref = torch.zeros_like(cut, dtype=torch.float64)
    for i, n in enumerate((200, 160)):
        for r in range(q):
            row = dict(c, q=c["q"][i * q + r:i * q + r + 1], table=c["table"][i:i + 1], start=torch.tensor([0, 1]),
                       seq=torch.tensor([min(n - q + r + 1, 40)]))
            o, vmax = K.attention(row["q"], c["cache"], 16, c["scales"], row["table"], row["start"], row["seq"], c["scale"])
            ref[i * q + r] = o[0]
            assert ((cut[i * q + r].double() - o[0]).abs() <= tolerance(o[0], vmax[0], cut.dtype)).all()


@pytest.mark.gpu
def test_attention_rows_outside_the_starts_are_left(ext, cuda_device):
    c = attention_case([(2, 40), (3, 50)], 4, 2, 64, 16, torch.float16)
    ref = run_attention(ext, cuda_device, c).cpu()
    q = torch.cat((c["q"], c["q"][:2]))
    got = run_attention(ext, cuda_device, dict(c, q=q)).cpu()
    assert torch.equal(got[:5], ref) and (got[5:] == 77).all()


@pytest.mark.gpu
def test_attention_page_numbers_are_clamped(ext, cuda_device):
    """Page numbers that no cache has must not read outside it."""
    c = attention_case([(1, 100), (150, 170)], 4, 2, 64, 16, torch.float16, stale=0)
    c["table"][0, 2], c["table"][1, 3] = 1 << 30, -5
    low = dict(c, table=c["table"].clone())
    low["table"][0, 2], low["table"][1, 3] = c["cache"].shape[0] - 1, 0
    assert torch.equal(run_attention(ext, cuda_device, c).cpu(), run_attention(ext, cuda_device, low).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("q,hq,hkv", [(1, 8, 2), (140, 8, 2), (600, 64, 16)])
def test_attention_other_stream_and_graph(ext, cuda_device, q, hq, hkv):
    c = {k: (v.to(cuda_device) if torch.is_tensor(v) else v) for k, v in
         attention_case([(q, 900), (q, max(q, 150))], hq, hkv, 128, 16, torch.float16).items()}
    ref = run_attention(ext, cuda_device, c)
    out = torch.zeros_like(ref)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            run_attention(ext, cuda_device, c, out=out)
        for _ in range(3):
            g.replay()
    st.synchronize()
    assert torch.equal(out, ref)


@pytest.mark.gpu
def test_attention_wrong_tensors(ext, cuda_device):
    c = {k: (v.to(cuda_device) if torch.is_tensor(v) else v) for k, v in
         attention_case([(1, 20), (1, 30)], 4, 2, 64, 16, torch.float16).items()}
    run_attention(ext, cuda_device, c)
    for bad in [dict(q=c["q"].float()), dict(q=c["q"][:, :3]), dict(table=c["table"].long()), dict(table=c["table"][:1]),
                dict(start=c["start"][:2]), dict(seq=c["seq"].long()), dict(scales=c["scales"].double()), dict(page=32),
                dict(scale=0.0), dict(max_q=-1), dict(cache=c["cache"][..., :-16])]:
        with pytest.raises(RuntimeError):
            run_attention(ext, cuda_device, {**c, **bad}, out=torch.zeros_like(c["q"]) if "q" not in bad else None)
    with pytest.raises(RuntimeError):
        run_attention(ext, cuda_device, c, out=torch.zeros_like(c["q"])[:1])


@pytest.mark.gpu
def test_attention_no_wait_gave_up(cuda_device):
    count = ctypes.c_uint64(1)
    cabi.call("cek_kv4_timeouts", ctypes.byref(count))
    assert count.value == 0


# ---- many rows: every SM busy, CTAs in pairs -----------------------------------------

def attention_by_matrices(dev, c, window):
    """oracle attention as float64 matrix products on the GPU, for prompts that the row loop would take minutes for."""
    hq, d = c["q"].shape[1:]
    hkv = c["cache"].shape[1]
    out = torch.zeros(c["q"].shape, dtype=torch.float64, device=dev)
    vmax = torch.zeros(c["q"].shape[:2], dtype=torch.float64, device=dev)
    for i, n in enumerate(c["seq"].tolist()):
        a, b = c["start"][i].item(), c["start"][i + 1].item()
        if a == b:
            continue
        keys = torch.arange(n)
        slots = (c["table"][i].long()[keys // c["page"]] * c["page"] + keys % c["page"]).numpy()
        k, v = (torch.from_numpy(K.decode(c["cache"], c["page"], d, slots, part, c["scales"])).to(dev) for part in (0, 1))
        pos, keys = (n - (b - a) + torch.arange(b - a, device=dev))[:, None], keys.to(dev)[None]
        seen = (keys <= pos) & ((keys > pos - window) if window else True)
        for h in range(hq):
            s = c["q"][a:b, h].to(dev).double() @ k[:, h * hkv // hq].T * c["scale"]
            out[a:b, h] = torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v[:, h * hkv // hq]
            top = v[:, h * hkv // hq].abs().amax(-1)
            vmax[a:b, h] = torch.where(seen, top, 0.0).amax(-1)
    return out.cpu(), vmax.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("lens,hq,hkv,d,dt,window", [([(1201, 1201), (1100, 1333)], 32, 4, 128, "f16", 0),
                                                     ([(1201, 1300), (1100, 1100)], 32, 4, 128, "bf16", 300),
                                                     ([(700, 900), (513, 513), (640, 640)], 40, 40, 128, "f16", 0),
                                                     ([(1500, 1500)], 56, 8, 128, "bf16", 0),
                                                     ([(1201, 1201), (1100, 1333)], 16, 4, 256, "f16", 0),
                                                     ([(1300, 1301), (9, 700), (1100, 1100)], 20, 4, 256, "bf16", 77)])
def test_attention_many_rows(ext, cuda_device, lens, hq, hkv, d, dt, window, page):
    c = attention_case(lens, hq, hkv, d, page, DT[dt])
    got = run_attention(ext, cuda_device, c, window).cpu()
    ref, vmax = attention_by_matrices(cuda_device, c, window)
    assert ((got.double() - ref).abs() <= tolerance(ref, vmax, got.dtype)).all()
    assert torch.equal(got, run_attention(ext, cuda_device, c, window).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 1, 128), (32, 8, 128), (4, 1, 64), (16, 8, 256)])
def test_attention_one_prompt_among_single_tokens(ext, cuda_device, hq, hkv, d):
    """One long request decides the kernel; 600 short ones (some of nothing) around it."""
    gen = torch.Generator().manual_seed(7)
    short = torch.randint(0, 40, (600,), generator=gen).tolist()
    lens = [(1 if n else 0, n) for n in short]
    lens[311] = (777, 790)
    lens[599] = (5, 33)
    c = attention_case(lens, hq, hkv, d, 16, torch.bfloat16)
    got = run_attention(ext, cuda_device, c).cpu()
    ref, vmax = attention_by_matrices(cuda_device, c, 0)
    assert ((got.double() - ref).abs() <= tolerance(ref, vmax, got.dtype)).all()
    # the same in two calls: slices of the request arrays
    out = torch.full_like(got, 77.0, device=cuda_device)
    for part, longest in ((slice(0, 311), 1), (slice(311, 312), 777), (slice(312, 600), 5)):
        run_attention(ext, cuda_device, dict(c, table=c["table"][part], seq=c["seq"][part],
                                             start=c["start"][part.start:part.stop + 1]), max_q=longest, out=out)
    assert ((out.cpu().double() - ref).abs() <= tolerance(ref, vmax, got.dtype)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("longest", [60, 900])
def test_attention_more_requests_than_a_launch_takes(ext, cuda_device, longest):
    gen = torch.Generator().manual_seed(9)
    lens = [(0 if n % 7 == 0 else 1, n) for n in torch.randint(0, longest, (2500,), generator=gen).tolist()]
    c = attention_case(lens, 4, 2, 64, 32, torch.float16)
    got = run_attention(ext, cuda_device, c).cpu()
    ref, vmax = attention_by_matrices(cuda_device, c, 0)
    assert ((got.double() - ref).abs() <= tolerance(ref, vmax, got.dtype)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 100])
def test_attention_of_no_keys(ext, cuda_device, q):
    c = attention_case([(q, 0), (q, -4)], 4, 2, 64, 16, torch.float16)
    assert not run_attention(ext, cuda_device, c, max_seq=0).any()
    assert not run_attention(ext, cuda_device, c, max_seq=500).any()
    c["table"] = c["table"][:, :0]
    assert not run_attention(ext, cuda_device, c, max_seq=500).any()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 256])
def test_attention_many_rows_nan_stays_behind(ext, cuda_device, d):
    """A NaN value scale in each half of the channels, seen by the last rows of one head alone."""
    n, page = 1300, 16
    c = attention_case([(1201, n), (1100, 1100)], 32, 4, d, page, torch.float16)
    ref = run_attention(ext, cuda_device, c).cpu()
    off = K.offsets(page, d)
    nan = torch.zeros_like(ref, dtype=torch.bool)
    for key, group in ((n - 1, 1), (n - 7, d // 16 - 2)):
        c["cache"][c["table"][0, key // page].item(), 1, off[3] + (key % page) * (d // 16) + group] = 0x7F
        nan[1201 - (n - key):1201, 8:16, 16 * group:16 * group + 16] = True
    got = run_attention(ext, cuda_device, c).cpu()
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], ref[~nan])


# ---- keys of a few row blocks split over the SMs and joined ---------------------------

def split_case(hq, hkv, d, q, n, dt, page=64):
    """A chunk behind a long context, one behind a short one, one whose first rows stand before position 0."""
    return attention_case([(q, n), (q, n // 7), (q, 5)], hq, hkv, d, page, DT[dt])


def check_is_split(c):
    """Few row blocks against 148 SMs and 8 tiles and more: the pieces go through the workspace."""
    assert cabi.lib().cek_kv4_attention_workspace_bytes(len(c["seq"]), c["q"].shape[0], c["q"].shape[1], c["cache"].shape[1],
                                                        c["q"].shape[2], c["max_q"], c["max_seq"]) > 0


SPLIT = [(8, 1, 128, 10, 4097), (8, 1, 128, 40, 5000), (8, 2, 128, 140, 900), (4, 2, 256, 40, 4097), (4, 1, 256, 130, 5003),
         (4, 1, 64, 20, 4097), (8, 2, 64, 50, 6001)]  # one row block and two beside each other of each width


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,q,n", SPLIT)
@pytest.mark.parametrize("window", [0, 100, 2500])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_split_keys(ext, cuda_device, hq, hkv, d, q, n, window, dt):
    """With a window most pieces hold no tile."""
    c = split_case(hq, hkv, d, q, n, dt)
    check_is_split(c)
    got = run_attention(ext, cuda_device, c, window).cpu()
    ref, vmax = attention_by_matrices(cuda_device, c, window)
    ref = ref.nan_to_num()  # softmax over no keys
    assert ((got.double() - ref).abs() <= tolerance(ref, vmax, got.dtype)).all()
    assert not got[2 * q:3 * q - 5].any()
    assert torch.equal(got, run_attention(ext, cuda_device, c, window).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,q,n", SPLIT)
def test_attention_split_keys_nan(ext, cuda_device, hq, hkv, d, q, n):
    """NaN value scales: in a middle piece, for every row of a kv head, and near the end, for its last rows."""
    c = split_case(hq, hkv, d, q, n, "f16")
    check_is_split(c)
    ref = run_attention(ext, cuda_device, c).cpu()
    off, page, group, h = K.offsets(64, d), 64, hq // hkv, hkv - 1
    nan = torch.zeros_like(ref, dtype=torch.bool)
    for key, g16 in (((n - q) // 2, 1), (n - 3, d // 16 - 1)):
        c["cache"][c["table"][0, key // page].item(), h, off[3] + (key % page) * (d // 16) + g16] = 0x7F
        nan[max(0, key - (n - q)):q, h * group:(h + 1) * group, 16 * g16:16 * g16 + 16] = True
    got = run_attention(ext, cuda_device, c).cpu()
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], ref[~nan])


# ---- append and gather on both sides of the change to two units a thread ----------------

def near(dev, d, channels, blocks, hkv, more):
    """Tokens that fill `blocks` blocks an SM, the change's place, and `more`."""
    return 256 // (d // channels) * blocks * torch.cuda.get_device_properties(dev).multi_processor_count // hkv + more


@pytest.mark.gpu
@pytest.mark.parametrize("d,hkv,page,dt,aligned", [(64, 7, 16, "f16", True), (64, 32, 128, "bf16", False), (128, 8, 64, "bf16", True),
                                                   (128, 5, 32, "f16", False), (256, 3, 16, "f16", True), (256, 32, 64, "bf16", False)])
@pytest.mark.parametrize("more", [0, 1, 40])
def test_append_bits_long(ext, cuda_device, d, hkv, page, dt, aligned, more):
    """Tokens drawn from a pool whose codes the oracle gives; the last slots skipped, negative or past the cache."""
    dev, pool = cuda_device, 512
    T = near(dev, d, 16, 64, hkv, more)
    gen = torch.Generator().manual_seed(T)
    scales = scales_for(hkv, gen)
    k, v = (special((torch.randn(pool, hkv, d, generator=gen) * size).to(DT[dt])) for size in (1.0, 0.1))
    pick = torch.randint(0, pool, (T,), generator=gen)
    pages = -(-T // page) + 1
    slots = torch.randperm(pages * page, generator=gen)[:T]
    slots[-2], slots[-5], slots[T // 2] = -1, pages * page, -7
    ref = torch.zeros(pages, hkv, page_bytes(page, d), dtype=torch.uint8)
    off, ok = K.offsets(page, d), (slots >= 0) & (slots < pages * page)
    p, r = slots[ok] // page, slots[ok] % page
    for part, x in ((0, k), (1, v)):
        for start, width, what in zip(off[2 * part:], (d // 2, d // 16), K.quantize(x, scales[part])):
            ref[:, :, start:start + page * width].view(pages, hkv, page, width)[p, :, r] = what[pick[ok]]
    lead = 0 if aligned else 1
    wide = torch.zeros(T, hkv, d + 8, dtype=DT[dt], device=dev)
    wide[:, :, lead:lead + d] = k.to(dev)[pick.to(dev)]
    cache = torch.zeros_like(ref, device=dev)
    ext.esimd_kv4_append(wide[:, :, lead:lead + d], v.to(dev)[pick.to(dev)], scales.to(dev), slots.to(dev), cache, page)
    assert torch.equal(cache.cpu(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("d,hkv,page,dt,aligned", [(64, 32, 16, "bf16", True), (64, 7, 128, "f16", False), (128, 8, 64, "f16", True),
                                                   (128, 5, 32, "bf16", False), (256, 3, 16, "bf16", True), (256, 32, 64, "f16", False)])
@pytest.mark.parametrize("more", [0, 1, 40])
def test_gather_long(ext, cuda_device, d, hkv, page, dt, aligned, more):
    """Slots of a small cache read many times over; some near the end negative or past the cache."""
    dev, pages = cuda_device, 5
    T = near(dev, d, 8, 8, hkv, more)
    gen = torch.Generator().manual_seed(T)
    scales = scales_for(hkv, gen)
    cache = torch.randint(0, 256, (pages, hkv, page_bytes(page, d)), generator=gen, dtype=torch.uint8)
    slots = torch.randint(0, pages * page, (T,), generator=gen)
    slots[-1], slots[-4], slots[T // 2] = pages * page, -1, -9
    ok = ((slots >= 0) & (slots < pages * page))[:, None, None]
    lead = 0 if aligned else 1
    wide = torch.full((2, T, hkv, d + 8), 7.0, dtype=DT[dt], device=dev)
    out = wide[:, :, :, lead:lead + d]
    ext.esimd_kv4_gather(cache.to(dev), scales.to(dev), slots.to(dev), out[0], out[1], page)
    for part in (0, 1):
        values = torch.from_numpy(K.decode(cache, page, d, torch.arange(pages * page).numpy(), part, scales)).float().to(DT[dt])
        ref = torch.where(ok, values[slots.clamp(0, pages * page - 1)], torch.zeros((), dtype=DT[dt]))
        assert torch.equal(torch.nan_to_num(out[part].cpu(), 1234.0), torch.nan_to_num(ref, 1234.0))
    assert (wide[..., :lead] == 7).all() and (wide[..., lead + d:] == 7).all()


# ---- numbers at the end of 32 bits ------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,q,n", [(2, 1, 64, 300, 150), (8, 1, 128, 200, 190), (4, 1, 256, 100, 70), (8, 2, 128, 4, 2),
                                          (1, 1, 64, 1, 9)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
def test_attention_window_beyond_any_length(ext, cuda_device, hq, hkv, d, q, n, window):
    """No window at all, also for a request whose first rows stand before position 0."""
    c = attention_case([(q, n), (q, 900)], hq, hkv, d, 16, torch.float16)
    assert torch.equal(run_attention(ext, cuda_device, c, window).cpu(), run_attention(ext, cuda_device, c).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [12, 16])
@pytest.mark.parametrize("c,n", [(2 ** 31 - 1, 1_200_000_000), (2 ** 31 - 2, 3), (2 ** 31 - 1, 0), (5, 2 ** 31 - 50)])
def test_plan_refuses_lengths_past_32_bits(ext, cuda_device, page, c, n):
    """A sum that would wrap is refused like any that its row cannot hold; the requests beside it are served."""
    got = run_plan(ext, cuda_device, [2, n, 1], [3, c, 5], [[7, 0], [0, 0], [8, 9]], [1, 2, 3], 3, page, 4)
    first = [7 * page + 3, 7 * page + 4]
    if n:
        pos, slots = [3, 4, c, c + 1], first + [-1, -1]
    else:
        pos, slots = [3, 4, 5, 0], first + [8 * page + 5, -1]
    assert got == ([[7, 0], [0, 0], [8, 9]], [0, 2, n + 2, n + 3], [5, ~c, 6], 3, pos, slots)


# ---- a cache without heads ---------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("heads", [0, 4])
def test_cache_without_heads_is_refused(ext, cuda_device, heads):
    i32 = dict(dtype=torch.int32, device=cuda_device)
    cache = torch.zeros(2, 0, page_bytes(16, 64), dtype=torch.uint8, device=cuda_device)
    scales = torch.ones(2, 0, device=cuda_device)
    q = torch.zeros(1, heads, 64, dtype=torch.float16, device=cuda_device)
    with pytest.raises(RuntimeError):
        ext.esimd_kv4_attention(q, cache, scales, torch.zeros(1, 1, **i32), torch.tensor([0, 1], **i32), torch.ones(1, **i32),
                                torch.zeros_like(q), 16, 0.125, 1, 16)
    kv, slots = q[:, :0], torch.zeros(1, dtype=torch.int64, device=cuda_device)
    with pytest.raises(RuntimeError):
        ext.esimd_kv4_append(kv, kv, scales, slots, cache, 16)
    with pytest.raises(RuntimeError):
        ext.esimd_kv4_gather(cache, scales, slots, kv, kv, 16)


# ---- counts at the end of 32 bits ----------------------------------------------------------

@pytest.mark.parametrize("kw", [dict(W=2 ** 27, ts=2 ** 27), dict(W=2 ** 60, ts=2 ** 60), dict(T=2 ** 31 - 1, mq=2 ** 31 - 1),
                                dict(T=2 ** 30, mq=2 ** 30, hq=8)])
def test_attention_refuses_counts_past_32_bits(kw):
    """Keys of a row of the table, rows of a kv head."""
    assert _attend(**{"ms": 2 ** 31 - 1, **kw}) == cabi.CEK_ERR_INVALID_ARG


def test_attention_refuses_more_tiles_than_it_counts():
    """65535 heads over 2^27 keys: 2^37 tiles of one request."""
    wide = dict(kv_heads=65535, page_stride=65535 * page_bytes(16, 64))
    assert _attend(_cache(**wide), hq=65535, W=2 ** 23, ts=2 ** 23, ms=2 ** 27) == cabi.CEK_ERR_INVALID_ARG
    assert _attend(_cache(**wide), hq=65535, B=0) == cabi.CEK_OK


@pytest.mark.gpu
def test_attention_loose_bounds_in_several_launches(ext, cuda_device):
    """Tables so wide that the bound on tiles allows some 250 requests a launch; the lengths are short."""
    gen = torch.Generator().manual_seed(11)
    lens = [(0 if n % 7 == 0 else 1, n) for n in torch.randint(0, 700, (300,), generator=gen).tolist()]
    c = attention_case(lens, 16, 8, 64, 128, torch.float16)
    ref, vmax = attention_by_matrices(cuda_device, c, 0)
    table = torch.zeros(300, 130000, dtype=torch.int32, device=cuda_device)
    table[:, :c["table"].shape[1]] = c["table"].to(cuda_device)
    got = run_attention(ext, cuda_device, dict(c, table=table), max_seq=130000 * 128).cpu()
    assert ((got.double() - ref).abs() <= tolerance(ref, vmax, got.dtype)).all()
